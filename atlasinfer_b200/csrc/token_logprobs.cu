// Log probabilities of given tokens, the entropy of every row of logits, and its likeliest tokens, in one pass over the logits.
//
//   p_i = exp((l_i - m) / T) / S;   log p = (l - m) / T - log S;   H = log S - (sum e_i d_i) / (S T),  e_i = exp(d_i / T), d_i = l_i - m
//
// with the running maximum m of an online softmax (Milakov & Gimelshein 2018): every thread keeps m, S and the sum of e d, and
// they are joined at the end.  Differences come before products, so that l - m is exact for 16-bit logits and the error of a log
// probability does not grow with the logits themselves.
//
// The likeliest tokens cost nothing in that pass: the maxima of 32 groups of threads are known after it, and the k-th largest of
// those is at most the k-th largest logit.  Only threads whose own maximum reaches it look at their logits again (from L2), each
// warp for its own, and keep what is above the worst of a sorted list, one entry a lane: (logit, lowest index first) as one
// 64-bit key.  Lists are joined by bitonic merges (Batcher 1968).  A row of equal logits, or one with fewer than k that are not
// masked, is looked at twice; nothing has a fixed room that could overflow.
#include "rows.cuh"

namespace atlas {
namespace {

constexpr int LP_GROUPS = 32;
constexpr float LP_FLOOR = -1e28f;   // stands for smaller d where they are multiplied by e = 0: times 2^30 it is finite still

struct LogprobParams {
    const char *logits;
    const void *tokens;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_tokens;
    int64_t stride;      // bytes
    int vocab, top;
    float exponent, inverse_temperature;   // log2(e) / T, 1 / T
    bool wide_tokens;
};

template <int DTYPE>
struct Logits {
    static constexpr int SIZE = DTYPE == ATLAS_DTYPE_F32 ? 4 : 2, PER = 16 / SIZE;
    static __device__ __forceinline__ float at(const char *row, int i) {
        return DTYPE == ATLAS_DTYPE_F32 ? reinterpret_cast<const float *>(row)[i] : from16(reinterpret_cast<const uint16_t *>(row)[i], DTYPE == ATLAS_DTYPE_BF16);
    }
    // Piece j: the 16 bytes that begin at logit j PER - shift; what is not in the row is -inf.
    static __device__ __forceinline__ void piece(const char *row, int first, int vocab, float (&f)[PER]) {
        if (first >= 0 && first + PER <= vocab) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row + (int64_t)first * SIZE));
            if constexpr (DTYPE == ATLAS_DTYPE_F32) {
                f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
            } else {
                open16<DTYPE == ATLAS_DTYPE_BF16>(v, f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) f[i] = first + i >= 0 && first + i < vocab ? at(row, first + i) : -INFINITY;
        }
    }
};

__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Maximum, sum of e and sum of e d of some logits; the maximum of none is -inf, and then d is taken from 0.
struct Stats {
    float m, s, t;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void move_to(Stats &a, float m, float exponent) {
    const float d = a.m == -INFINITY ? 0.f : a.m - m, f = exp2_of(d * exponent);
    a.t = f * (a.t + a.s * fmaxf(d, LP_FLOOR));
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ Stats joined(Stats a, Stats b, float exponent) {
    const float m = fmaxf(a.m, b.m);
    move_to(a, m, exponent);
    move_to(b, m, exponent);
    return {m, a.s + b.s, a.t + b.t};
}

// Larger for larger logits (NaN above all, -0 as 0), for equal ones larger for the lower index; never 0.
__device__ __forceinline__ unsigned long long key_of(float l, int index) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    const uint32_t o = l != l ? 0xffffffffu : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return (unsigned long long)o << 32 | (uint32_t)~index;
}
// The 32 largest of two lists that lie over the lanes in descending order, in descending order.
__device__ __forceinline__ unsigned long long merged(unsigned long long a, unsigned long long b, int lane) {
    const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = a > r ? a : r;
#pragma unroll
    for (int k = 16; k; k /= 2) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, a, k);
        a = ((lane & k) == 0) == (a > o) ? a : o;
    }
    return a;
}

// A row is a CTA's.
template <int DTYPE, int THREADS>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const LogprobParams p) {
    using L = Logits<DTYPE>;
    constexpr int WARPS = THREADS / 32, PER = L::PER, AHEAD = 4, GROUP = THREADS / LP_GROUPS;
    __shared__ Stats stats[WARPS];
    __shared__ float group_max[LP_GROUPS];
    __shared__ unsigned long long lists[WARPS][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    wait_for_front();
    const int64_t row_at = blockIdx.x;
    const char *row = p.logits + row_at * p.stride;
    const int shift = (int)(((uintptr_t)row & 15) / L::SIZE), pieces = (p.vocab + shift + PER - 1) / PER;

    // ---- one pass: maximum and sums ----------------------------------------------------------------------
    Stats mine = {-INFINITY, 0.f, 0.f};
    for (int j0 = tid; j0 < pieces; j0 += AHEAD * THREADS) {
        float f[AHEAD][PER];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int j = j0 + a * THREADS;
            if (j < pieces) {
                L::piece(row, j * PER - shift, p.vocab, f[a]);
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i) f[a][i] = -INFINITY;
            }
        }
        float m = mine.m;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int i = 0; i < PER; ++i) m = fmaxf(m, f[a][i]);
        if (m > mine.m) move_to(mine, m, p.exponent);
        const float base = base_of(m);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float d = f[a][i] - base, e = exp2_of(d * p.exponent);
                mine.s += e;
                mine.t += e * fmaxf(d, LP_FLOOR);
            }
    }
    const float own = mine.m;
    const bool odd = mine.s != mine.s;   // NaN or +inf among them
    Stats all = mine;
#pragma unroll
    for (int k = 16; k; k /= 2) {
        const Stats o = {__shfl_xor_sync(0xffffffffu, all.m, k), __shfl_xor_sync(0xffffffffu, all.s, k), __shfl_xor_sync(0xffffffffu, all.t, k)};
        all = joined(all, o, p.exponent);
    }
    float group = own;
#pragma unroll
    for (int k = GROUP / 2; k; k /= 2) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, k));
    if (lane == 0) stats[warp] = all;
    if (tid % GROUP == 0) group_max[tid / GROUP] = group;
    __syncthreads();

    // ---- the likeliest -----------------------------------------------------------------------------------
    unsigned long long list = 0;
    if (p.top) {
        const float g = group_max[lane];
        int rank = 0;
#pragma unroll
        for (int k = 0; k < LP_GROUPS; ++k) {
            const float o = __shfl_sync(0xffffffffu, g, k);
            rank += o > g || (o == g && k < lane);
        }
        const float least = __shfl_sync(0xffffffffu, g, __ffs(__ballot_sync(0xffffffffu, rank == p.top - 1)) - 1);
        unsigned owners = __ballot_sync(0xffffffffu, own >= least || odd);
        const int steps = (pieces + THREADS - 1) / THREADS;
        while (owners) {
            const int who = warp * 32 + __ffs(owners) - 1;
            owners &= owners - 1;
            for (int s0 = 0; s0 < steps; s0 += 32) {   // the warp reads that thread's pieces, one a lane
                const int j = who + (s0 + lane) * THREADS, first = j * PER - shift;
                const bool live = s0 + lane < steps && j < pieces;
                float f[PER];
                if (live) L::piece(row, first, p.vocab, f);
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    unsigned long long key = 0;
                    if (live && first + i >= 0 && first + i < p.vocab && !(f[i] < least)) key = key_of(f[i], first + i);
                    while (true) {
                        const unsigned better = __ballot_sync(0xffffffffu, key > __shfl_sync(0xffffffffu, list, p.top - 1));
                        if (!better) break;
                        const int from = __ffs(better) - 1;
                        const unsigned long long k = __shfl_sync(0xffffffffu, key, from);
                        if (lane == from) key = 0;
                        const unsigned long long before = __shfl_up_sync(0xffffffffu, list, 1);
                        const bool behind = list < k;
                        list = !behind ? list : lane == 0 || before >= k ? k : before;
                    }
                }
            }
        }
        lists[warp][lane] = list;
#pragma unroll
        for (int half = WARPS / 2; half; half /= 2) {
            __syncthreads();
            if (warp < half) lists[warp][lane] = list = merged(list, lists[warp + half][lane], lane);
        }
    }
    if (warp) return;

    // ---- the answer --------------------------------------------------------------------------------------
    all = lane < WARPS ? stats[lane] : Stats{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int k = 16; k; k /= 2) {
        const Stats o = {__shfl_xor_sync(0xffffffffu, all.m, k), __shfl_xor_sync(0xffffffffu, all.s, k), __shfl_xor_sync(0xffffffffu, all.t, k)};
        all = joined(all, o, p.exponent);
    }
    const float log_sum = logf(all.s);
    auto log_chance = [&](float l) { return all.s == 0.f ? -INFINITY : (l - all.m) * p.inverse_temperature - log_sum; };
    if (lane == 0) {
        const int64_t token = p.wide_tokens ? reinterpret_cast<const int64_t *>(p.tokens)[row_at] : reinterpret_cast<const int32_t *>(p.tokens)[row_at];
        p.logprobs[row_at] = token < 0 ? 0.f : token >= p.vocab ? NAN : log_chance(L::at(row, (int)token));
        const float h = log_sum - all.t / all.s * p.inverse_temperature;
        p.entropy[row_at] = all.s == 0.f || h < 0.f ? 0.f : h;
    }
    if (lane < p.top) {
        const int index = (int)~(uint32_t)list;
        p.top_tokens[row_at * p.top + lane] = index;
        p.top_logprobs[row_at * p.top + lane] = log_chance(L::at(row, index));
    }
}

template <int DTYPE>
int launch(const LogprobParams &p, int64_t rows, cudaStream_t st, const char *what) {
    return launch_early(token_logprobs_kernel<DTYPE, 512>, dim3((unsigned)rows), 512, 0, st, what, p);
}

}  // namespace
}  // namespace atlas

extern "C" int atlas_token_logprobs(const AtlasTokenLogprobs *q, void *stream) {
    using namespace atlas;
    clear_error();
    const char *what = "atlas_token_logprobs";
    ATLAS_RETURN_IF(!q, ATLAS_ERR_BAD_ARGUMENT, "%s: no arguments", what);
    ATLAS_RETURN_IF(q->dtype < ATLAS_DTYPE_F16 || q->dtype > ATLAS_DTYPE_F32, ATLAS_ERR_BAD_ARGUMENT, "%s: dtype %d", what, q->dtype);
    ATLAS_RETURN_IF(q->rows < 0 || q->vocab < 1, ATLAS_ERR_BAD_ARGUMENT, "%s: %lld rows of %lld", what, (long long)q->rows, (long long)q->vocab);
    ATLAS_RETURN_IF(q->rows > 0x7fffffff || q->vocab > (1 << 30), ATLAS_ERR_UNSUPPORTED, "%s: %lld rows of %lld", what, (long long)q->rows, (long long)q->vocab);
    ATLAS_RETURN_IF(q->top < 0 || q->top > q->vocab, ATLAS_ERR_BAD_ARGUMENT, "%s: the top %d of %lld", what, q->top, (long long)q->vocab);
    ATLAS_RETURN_IF(q->top > ATLAS_LOGPROBS_MAX_TOP, ATLAS_ERR_UNSUPPORTED, "%s: top %d is more than %d", what, q->top, ATLAS_LOGPROBS_MAX_TOP);
    ATLAS_RETURN_IF(!(q->temperature >= 1e-4f && q->temperature <= 1e4f), ATLAS_ERR_BAD_ARGUMENT, "%s: temperature %g", what, (double)q->temperature);
    ATLAS_RETURN_IF(q->token_bytes != 4 && q->token_bytes != 8, ATLAS_ERR_BAD_ARGUMENT, "%s: tokens of %d bytes", what, q->token_bytes);
    if (q->rows == 0) return ATLAS_OK;
    ATLAS_RETURN_IF(!q->logits || !q->tokens || !q->logprobs || !q->entropy || (q->top && (!q->top_tokens || !q->top_logprobs)), ATLAS_ERR_BAD_ARGUMENT,
                    "%s: null pointer", what);
    const int size = q->dtype == ATLAS_DTYPE_F32 ? 4 : 2;
    ATLAS_RETURN_IF((uintptr_t)q->logits % size || (uintptr_t)q->tokens % q->token_bytes, ATLAS_ERR_BAD_ARGUMENT, "%s: a buffer is not aligned to its type", what);
    const int dev = check_device();
    if (dev != ATLAS_OK) return dev;
    LogprobParams p = {};
    p.logits = (const char *)q->logits, p.tokens = q->tokens;
    p.logprobs = q->logprobs, p.entropy = q->entropy, p.top_tokens = q->top_tokens, p.top_logprobs = q->top_logprobs;
    p.stride = q->logits_stride * size, p.vocab = (int)q->vocab, p.top = q->top;
    p.exponent = (float)(1.4426950408889634 / q->temperature), p.inverse_temperature = (float)(1.0 / q->temperature);
    p.wide_tokens = q->token_bytes == 8;
    cudaStream_t st = (cudaStream_t)stream;
    return q->dtype == ATLAS_DTYPE_F32 ? launch<ATLAS_DTYPE_F32>(p, q->rows, st, what)
           : q->dtype == ATLAS_DTYPE_BF16 ? launch<ATLAS_DTYPE_BF16>(p, q->rows, st, what) : launch<ATLAS_DTYPE_F16>(p, q->rows, st, what);
}
