// Log probabilities of given tokens, the entropy of every row of logits, and its likeliest tokens, in one pass over the logits.
//
//   p_i = exp((l_i - m) / T) / S;   log p = (l - m) / T - log S;   H = log S - (sum e_i d_i) / (S T),  e_i = exp(d_i / T), d_i = l_i - m
//
// with the running maximum m of an online softmax (Milakov & Gimelshein 2018): every thread keeps m, S and the sum of e d, and
// they are joined at the end.  Differences come before products, so that l - m is exact for 16-bit logits and the error of a log
// probability does not grow with the logits themselves.
//
// The likeliest tokens cost nothing in that pass: the maxima of 64 groups of threads are known after it, and the k-th largest of
// those is at most the k-th largest logit.  Only threads whose own maximum reaches it look again, at the batch that holds it (at
// all of theirs if more than one batch reaches it); what reaches it
// (k and a few more) is collected as 64-bit keys (logit, lowest index first), and the place of a key is the number of keys
// above it.  Where far more reach it (rows of equal logits) the k-th largest key of some of them is a higher floor for another
// look, which at least 224 keys fewer reach: looks in proportion to the vocabulary, if the largest logits ascend with their index and lie
// in the pieces of fewer than k of the groups.  Such a row costs more than one of drawn logits (32 tokens, us: 1 x 50272 fp32 23
// instead of 12, 1 x 262144 50 instead of 14, 64 x 262144 375 instead of 18, 400 x 262144 6550 instead of 77); a row that ascends
// as a whole 20 to 41 instead of 11 to 20 at 50272.  No two keys are equal, so the answer does not depend on the order in which they are found.
#include <algorithm>

#include "rows.cuh"

namespace atlas {
namespace {

constexpr int LP_GROUPS = 64;
constexpr int LP_MAX_PARTS = 8;      // CTAs of a row: a power of two, the portable cluster size
constexpr float LP_FLOOR = -1e28f;   // stands for smaller d where they are multiplied by e = 0: times 2^30 it is finite still

struct LogprobParams {
    const char *logits;
    const void *tokens;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_tokens;
    int64_t stride;      // bytes
    int vocab, top, parts;
    float exponent, inverse_temperature;   // log2(e) / T, 1 / T
    bool wide_tokens;
};

// Two fp32 numbers that are worked on by one instruction.
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair_of(float lo, float hi) {
    pair_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float low(pair_t v) {
    float r;
    asm("{.reg .f32 h; mov.b64 {%0, h}, %1;}" : "=f"(r) : "l"(v));
    return r;
}
__device__ __forceinline__ float high(pair_t v) {
    float r;
    asm("{.reg .f32 l; mov.b64 {l, %0}, %1;}" : "=f"(r) : "l"(v));
    return r;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
    pair_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
    pair_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
    pair_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A piece is 16 aligned bytes of a row; a batch is so many of a thread's.
constexpr int batch_pieces(int dtype) { return dtype == ATLAS_DTYPE_F32 ? 4 : 3; }
template <int DTYPE>
struct Logits {
    static constexpr bool WIDE = DTYPE == ATLAS_DTYPE_F32, BF16 = DTYPE == ATLAS_DTYPE_BF16;
    static constexpr int SIZE = WIDE ? 4 : 2, PER = 16 / SIZE;
    static constexpr uint32_t NONE = WIDE ? 0xff800000u : BF16 ? 0xff80ff80u : 0xfc00fc00u;   // -inf
    static __device__ __forceinline__ float at(const char *row, int i) {
        return WIDE ? reinterpret_cast<const float *>(row)[i] : from16(reinterpret_cast<const uint16_t *>(row)[i], BF16);
    }
    // The piece that begins at logit `first`; what is not in the row is -inf.
    static __device__ __forceinline__ uint4 piece(const char *row, int first, int vocab) {
        if (first >= 0 && first + PER <= vocab) return __ldg(reinterpret_cast<const uint4 *>(row + (int64_t)first * SIZE));
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = NONE;
            if (WIDE) {
                if (first + i >= 0 && first + i < vocab) w[i] = __ldg(reinterpret_cast<const uint32_t *>(row) + first + i);
            } else {
                const int k = first + 2 * i;
                if (k >= 0 && k < vocab) w[i] = (w[i] & 0xffff0000u) | __ldg(reinterpret_cast<const uint16_t *>(row) + k);
                if (k + 1 >= 0 && k + 1 < vocab) w[i] = (w[i] & 0xffffu) | (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(row) + k + 1) << 16;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static constexpr float LOWEST = DTYPE == ATLAS_DTYPE_F16 ? -65504.f : BF16 ? -0x1.fep127f : -0x1.fffffep127f;
    // -inf becomes the lowest finite number (NaN stays).
    static __device__ __forceinline__ uint4 finite(const uint4 &v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (WIDE) r[i] = __float_as_uint(max_or_nan(__uint_as_float(w[i]), LOWEST));
            else if (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(w[i]), "r"(0xff7fff7fu));
            else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(w[i]), "r"(0xfbfffbffu));
        }
        return make_uint4(r[0], r[1], r[2], r[3]);
    }
    // Whether all of some pieces is -inf.
    template <int N>
    static __device__ __forceinline__ bool masked(const uint4 (&v)[N]) {
        uint32_t other = 0;
#pragma unroll
        for (int a = 0; a < N; ++a) other |= (v[a].x ^ NONE) | (v[a].y ^ NONE) | (v[a].z ^ NONE) | (v[a].w ^ NONE);
        return other == 0;
    }
    // Its logits, two by two.
    static constexpr int PAIRS = PER / 2;
    static __device__ __forceinline__ pair_t pair(const uint4 &v, int i) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if (WIDE) return pair_of(__uint_as_float(w[2 * i % 4]), __uint_as_float(w[(2 * i + 1) % 4]));
        if (BF16) return pair_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        return pair_of(f.x, f.y);
    }
    // The largest of `m` and of some pieces (NaN is passed over).
    template <int N>
    static __device__ __forceinline__ float most(float m, const uint4 (&v)[N]) {
        if (WIDE) {
#pragma unroll
            for (int a = 0; a < N; ++a) {
                const uint32_t w[4] = {v[a].x, v[a].y, v[a].z, v[a].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(w[i]));
            }
            return m;
        }
        uint32_t most2 = NONE;
#pragma unroll
        for (int a = 0; a < N; ++a) {
            const uint32_t w[4] = {v[a].x, v[a].y, v[a].z, v[a].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (BF16) asm("max.bf16x2 %0, %0, %1;" : "+r"(most2) : "r"(w[i]));
                else asm("max.f16x2 %0, %0, %1;" : "+r"(most2) : "r"(w[i]));
            }
        }
        const pair_t p = pair(make_uint4(most2, most2, most2, most2), 0);
        return fmaxf(m, fmaxf(low(p), high(p)));
    }
};

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
__device__ __forceinline__ float logit_of(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o >> 31) ? o ^ 0x80000000u : ~o);
}
// A number for each lane that comes here, from a counter in shared memory; lanes that come together take theirs together.
__device__ __forceinline__ int place_in(int *counter, int lane) {
    const unsigned here = __activemask();
    const int leader = __ffs(here) - 1;
    int n = 0;
    if (lane == leader) n = atomicAdd(counter, __popc(here));
    return __shfl_sync(here, n, leader) + __popc(here & ((1u << lane) - 1));
}
// How many of some keys are above one.
__device__ __forceinline__ int above(const unsigned long long *keys, int count, unsigned long long key) {
    int n = 0;
#pragma unroll 8
    for (int k = 0; k < count; ++k) n += keys[k] > key;
    return n;
}
// This lane's number where the 32 of a warp lie in descending order over its lanes (Batcher 1968).
__device__ __forceinline__ float sorted(float v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int k = size / 2; k; k /= 2) {
            const float o = __shfl_xor_sync(0xffffffffu, v, k);
            v = ((lane & k) == 0) == ((lane & size) == 0 || size == 32) ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}
// A bound for the k-th largest of 64 numbers, two a lane, that is at most as large: up to 16 that of the 32 lanes' larger ones, which
// is found by one sort and seldom much smaller; above that the number itself (the 32 largest are the larger ones of one half
// in descending and the other in ascending order).
__device__ __forceinline__ float kth_largest(float a, float b, int k, int lane) {
    if (k <= 16) return __shfl_sync(0xffffffffu, sorted(fmaxf(a, b), lane), k - 1);
    a = sorted(a, lane), b = sorted(b, lane);
    a = fmaxf(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
    for (int d = 16; d; d /= 2) {
        const float o = __shfl_xor_sync(0xffffffffu, a, d);
        a = lane & d ? fminf(a, o) : fmaxf(a, o);
    }
    return __shfl_sync(0xffffffffu, a, k - 1);
}
template <typename T>
__device__ __forceinline__ T of_cta(const T &there, int rank) {   // the same place of another CTA of the cluster
    static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
    uint32_t at = (uint32_t)__cvta_generic_to_shared(&there);
    asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
    T v;
    if constexpr (sizeof(T) == 4) {
        uint32_t b;
        asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(b) : "r"(at) : "memory");
        v = *reinterpret_cast<T *>(&b);
    } else {
        unsigned long long b;
        asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(b) : "r"(at) : "memory");
        v = *reinterpret_cast<T *>(&b);
    }
    return v;
}
__device__ __forceinline__ Stats over_lanes(Stats all, int lanes, float exponent) {
    for (int k = lanes / 2; k; k /= 2) {
        const Stats o = {__shfl_xor_sync(0xffffffffu, all.m, k), __shfl_xor_sync(0xffffffffu, all.s, k), __shfl_xor_sync(0xffffffffu, all.t, k)};
        all = joined(all, o, exponent);
    }
    return all;
}

// A row is a cluster's of p.parts CTAs, each of which has a run of its pieces.
// SLOTS: batches of a thread that travel through shared memory (one of them may be the one in use), or 0: two, through registers.
template <int DTYPE, int THREADS, int SLOTS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const LogprobParams p) {
    using L = Logits<DTYPE>;
    constexpr int WARPS = THREADS / 32, PER = L::PER, AHEAD = batch_pieces(DTYPE), GROUP = THREADS / LP_GROUPS;
    __shared__ Stats stats[WARPS], together;
    __shared__ float group_max[LP_GROUPS];
    constexpr int CANDIDATES = 512;
    static_assert(CANDIDATES >= LP_MAX_PARTS * 32 && CANDIDATES / 2 > ATLAS_LOGPROBS_MAX_TOP, "room for the list of each CTA; floors rise");
    __shared__ unsigned long long candidates[CANDIDATES], list[32], raised;
    __shared__ int owners[THREADS], batch_count, full_count, candidate_count;   // (two lists, from either end)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x % p.parts;
    if (tid < 32) list[tid] = 0;
    if (tid == 0) batch_count = full_count = candidate_count = 0;
    wait_for_front();
    const int64_t row_at = blockIdx.x / p.parts;
    const char *row = p.logits + row_at * p.stride;
    const int shift = (int)(((uintptr_t)row & 15) / L::SIZE), every = (p.vocab + shift + PER - 1) / PER;
    const int begin = (int)((int64_t)every * rank / p.parts), pieces = (int)((int64_t)every * (rank + 1) / p.parts) - begin;
    const int at0 = begin * PER - shift;   // the first logit of this CTA's first piece
    int64_t token = 0;
    float given = 0.f;   // (asked for now, so that nobody waits for it at the end)
    if (rank == 0 && tid == 0) {
        token = p.wide_tokens ? reinterpret_cast<const int64_t *>(p.tokens)[row_at] : reinterpret_cast<const int32_t *>(p.tokens)[row_at];
        if (token >= 0 && token < p.vocab) given = L::at(row, (int)token);
    }

    // ---- one pass: maximum and sums ----------------------------------------------------------------------
    // pieces that lie in the row as a whole; of the others (the first or the last one of the row, or both) thread 0 takes care
    const int front = pieces > 0 && at0 < 0, whole = pieces - front - (at0 + pieces * PER > p.vocab && pieces > front);
    float most = -INFINITY, second = -INFINITY;   // of this thread's logits; of those outside of the batch with the largest
    int best = 0, batches = 0;                    // that batch
    pair_t sum = 0, weighted = 0;   // of e, of e d
    const pair_t exponent = pair_of(p.exponent, p.exponent);
    auto add_up = [&](const uint4 (&raw)[AHEAD]) {
        const float here = L::most(-INFINITY, raw), m = fmaxf(most, here);
        second = fmaxf(second, fminf(most, here));
        if (m > most) {
            best = batches;
            const float d = most == -INFINITY ? 0.f : most - m, f = exp2_of(d * p.exponent), g = fmaxf(d, LP_FLOOR);
            weighted = mul2(pair_of(f, f), fma2(sum, pair_of(g, g), weighted));
            sum = mul2(pair_of(f, f), sum);
            most = m;
        }
        const float base = base_of(m);
        const pair_t minus = pair_of(-base, -base);
        if (m < 1e30f && (L::LOWEST - m) * p.exponent < -160.f) {
            // what is as low as the type reaches has e = 0, and -inf may be taken as that: no product with d = -inf
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                for (int i = 0; i < L::PAIRS; ++i) {
                    const pair_t d = add2(L::pair(L::finite(raw[a]), i), minus), z = mul2(d, exponent);
                    const pair_t e = pair_of(exp2_of(low(z)), exp2_of(high(z)));
                    sum = add2(sum, e);
                    weighted = fma2(e, d, weighted);
                }
        } else if (!L::masked(raw)) {   // nothing but masked logits before this batch, or logits near the ends of their type
#pragma unroll 1
            for (int a = 0; a < AHEAD; ++a) {
                uint4 v = raw[0];
#pragma unroll
                for (int k = 1; k < AHEAD; ++k)
                    if (a == k) v = raw[k];
#pragma unroll
                for (int i = 0; i < L::PAIRS; ++i) {
                    const pair_t d = add2(L::pair(v, i), minus), z = mul2(d, exponent);
                    const pair_t e = pair_of(exp2_of(low(z)), exp2_of(high(z)));
                    sum = add2(sum, e);
                    weighted = fma2(e, pair_of(fmaxf(low(d), LP_FLOOR), fmaxf(high(d), LP_FLOOR)), weighted);
                }
            }
        }
        ++batches;
    };
    const uint4 none = make_uint4(L::NONE, L::NONE, L::NONE, L::NONE);
    const uint4 *next = reinterpret_cast<const uint4 *>(row + (int64_t)(at0 + front * PER) * L::SIZE) + tid;
    int left = whole > tid ? (whole - tid + THREADS - 1) / THREADS : 0;   // of this thread's pieces
    auto load = [&](uint4 (&to)[AHEAD]) {
        if (left >= AHEAD) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) to[a] = __ldg(next + a * THREADS);
        } else {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) to[a] = a < left ? __ldg(next + a * THREADS) : none;
        }
        next += AHEAD * THREADS;
        left -= AHEAD;
    };
    uint4 even[AHEAD];
    if constexpr (SLOTS > 0) {   // every thread's batches have places of their own: nothing but the thread waits for them
        extern __shared__ uint4 ring[];   // [SLOTS][AHEAD][THREADS]
        const uint32_t mine_at = (uint32_t)__cvta_generic_to_shared(ring + tid);
        auto fetch = [&](int slot) {
            auto one = [&](int a) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine_at + (slot * AHEAD + a) * THREADS * 16), "l"(next + a * THREADS) : "memory");
            };
            if (left >= AHEAD) {
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) one(a);
            } else {
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
                    if (a < left) one(a);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            next += AHEAD * THREADS;
            left -= AHEAD;
        };
        int rest = left, from = 0, to = SLOTS - 1;
#pragma unroll
        for (int s = 0; s < SLOTS - 1; ++s) fetch(s);
        for (; rest >= AHEAD; rest -= AHEAD) {
            asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 2) : "memory");
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) even[a] = ring[(from * AHEAD + a) * THREADS + tid];
            fetch(to);   // (where the batch before this one was: it has been used)
            add_up(even);
            from = from + 1 == SLOTS ? 0 : from + 1, to = to + 1 == SLOTS ? 0 : to + 1;
        }
        if (rest > 0) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) even[a] = a < rest ? ring[(from * AHEAD + a) * THREADS + tid] : none;
            add_up(even);
        }
    } else if (left > 0) {
        uint4 odds[AHEAD];   // one batch travels while the other one is summed up
        load(even);
        while (true) {
            bool more = left > 0;
            if (more) load(odds);
            add_up(even);
            if (!more) break;
            more = left > 0;
            if (more) load(even);
            add_up(odds);
            if (!more) break;
        }
    }
    if (tid == 0 && whole < pieces) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) even[a] = none;
        if (front) even[0] = L::piece(row, at0, p.vocab);
        if (front + whole < pieces) even[1] = L::piece(row, at0 + (pieces - 1) * PER, p.vocab);
        add_up(even);
        second = most;   // (this batch is none of three pieces in a row)
    }
    const Stats mine = {most, low(sum) + high(sum), low(weighted) + high(weighted)};
    const float own = mine.m;
    const bool odd = mine.s != mine.s;   // NaN or +inf among them
    Stats all = over_lanes(mine, 32, p.exponent);
    float group = own;
#pragma unroll
    for (int k = GROUP / 2; k; k /= 2) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, k));
    if (lane == 0) stats[warp] = all;
    if (tid % GROUP == 0) group_max[tid / GROUP] = group;
    __syncthreads();

    // ---- the likeliest -----------------------------------------------------------------------------------
    if (p.top) {
        const float bound = kth_largest(group_max[lane], group_max[lane + 32], p.top, lane);
        const int begins = max(0, at0), ends = min(p.vocab, at0 + pieces * PER);   // this CTA's logits
        // no key with this logit is smaller; where it is -inf, as many as are wanted reach that of the last one of the first so many
        unsigned long long floor = key_of(bound, 0) & 0xffffffff00000000ull;
        if (bound == -INFINITY && ends - begins >= p.top) floor = key_of(-INFINITY, begins + p.top - 1);
        const unsigned long long mine_at_most = odd ? ~0ull : key_of(own, max(0, at0 + (tid ? front + tid : 0) * PER));
        const int steps = (whole + THREADS - 1) / THREADS + 2;   // (the last two: what thread 0 took care of)
        while (true) {
            const float least = logit_of(floor);
            // a thread whose other batches do not reach the floor has candidates in one only
            if (mine_at_most >= floor) {
                if (odd || second >= least) owners[THREADS - 1 - place_in(&full_count, lane)] = tid;
                else owners[place_in(&batch_count, lane)] = best * THREADS + tid;
            }
            __syncthreads();
            const int of_batches = batch_count * AHEAD, items = of_batches + full_count * steps;
            // A candidate is a key that reaches the floor.  The order in which they are found does not matter: no two are equal.
            for (int item = tid; item < items && *(volatile int *)&candidate_count < CANDIDATES; item += THREADS) {
                int j;
                if (item < of_batches) {
                    const int owner = owners[item / AHEAD], batch = owner / THREADS;
                    j = front + owner % THREADS + (batch * AHEAD + item % AHEAD) * THREADS;
                    if (j >= front + whole) continue;
                } else {
                    const int step = (item - of_batches) / full_count, owner = owners[THREADS - 1 - (item - of_batches - step * full_count)];
                    j = front + owner + step * THREADS;
                    if (step >= steps - 2) {
                        if (owner || !(step == steps - 2 ? front : front + whole < pieces)) continue;
                        j = step == steps - 2 ? 0 : pieces - 1;
                    } else if (j >= front + whole) {
                        continue;
                    }
                }
                const int first = at0 + j * PER;
                const uint4 raw = L::piece(row, first, p.vocab);
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const pair_t l = L::pair(raw, i / 2);
                    const float v = i & 1 ? high(l) : low(l);
                    const int index = first + i;
                    if (!(v < least) && index >= 0 && index < p.vocab) {
                        const unsigned long long key = key_of(v, index);
                        if (key >= floor) {
                            const int n = place_in(&candidate_count, lane);
                            if (n < CANDIDATES) candidates[n] = key;
                        }
                    }
                }
            }
            __syncthreads();
            const int count = candidate_count;
            if (count < CANDIDATES) {   // all there are; the place of each is the number of those above it
                for (int c = tid; c < count; c += THREADS) {
                    const unsigned long long key = candidates[c];
                    const int place = above(candidates, count, key);
                    if (place < p.top) list[place] = key;
                }
                __syncthreads();
                break;
            }
            // Rows of equal logits, ascending ones: some of the candidates give a higher floor.
            for (int c = tid; c < CANDIDATES / 2; c += THREADS)
                if (above(candidates, CANDIDATES / 2, candidates[c]) == p.top - 1) raised = candidates[c];
            __syncthreads();
            floor = raised;
            if (tid == 0) batch_count = full_count = candidate_count = 0;
            __syncthreads();
        }
    }
    // ---- the CTAs of a row -------------------------------------------------------------------------------
    if (p.parts > 1) {
        if (warp == 0) {
            all = over_lanes(lane < WARPS ? stats[lane] : Stats{-INFINITY, 0.f, 0.f}, 32, p.exponent);
            if (lane == 0) together = all;
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank == 0) {
            if (p.top)
                for (int i = tid; i < p.parts * p.top; i += THREADS) candidates[i] = of_cta(list[i % p.top], i / p.top);
            if (warp == 0) all = lane < p.parts ? Stats{of_cta(together.m, lane), of_cta(together.s, lane), of_cta(together.t, lane)} : Stats{-INFINITY, 0.f, 0.f};
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // (nothing of the others is read any more)
        if (rank) return;
        if (p.top) {
            for (int c = tid; c < p.parts * p.top; c += THREADS) {
                const unsigned long long key = candidates[c];
                const int place = above(candidates, p.parts * p.top, key);
                if (place < p.top && key) list[place] = key;   // (a CTA of few logits has empty places)
            }
            __syncthreads();
        }
    }
    if (warp) return;

    // ---- the answer --------------------------------------------------------------------------------------
    all = p.parts > 1 ? over_lanes(all, 8, p.exponent) : over_lanes(lane < WARPS ? stats[lane] : Stats{-INFINITY, 0.f, 0.f}, 32, p.exponent);
    all = Stats{__shfl_sync(0xffffffffu, all.m, 0), __shfl_sync(0xffffffffu, all.s, 0), __shfl_sync(0xffffffffu, all.t, 0)};
    const float log_sum = logf(all.s);
    auto log_chance = [&](float l) { return all.s == 0.f ? -INFINITY : (l - all.m) * p.inverse_temperature - log_sum; };
    if (lane == 0) {
        p.logprobs[row_at] = token < 0 ? 0.f : token >= p.vocab ? NAN : log_chance(given);
        const float h = log_sum - all.t / all.s * p.inverse_temperature;
        p.entropy[row_at] = all.s == 0.f || h < 0.f ? 0.f : h;
    }
    if (lane < p.top) {
        p.top_tokens[row_at * p.top + lane] = (int)~(uint32_t)list[lane];
        p.top_logprobs[row_at * p.top + lane] = log_chance(logit_of(list[lane]));
    }
}

template <int DTYPE, int THREADS>
int launch_with(const LogprobParams &p, int64_t rows, cudaStream_t st, const char *what) {
    constexpr int SLOTS = Logits<DTYPE>::WIDE || THREADS == 512 ? 0 : 3;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * p.parts));
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = SLOTS * batch_pieces(DTYPE) * THREADS * 16;
    config.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.parts, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = p.parts > 1 ? 2 : 1;
    return check_cuda(cudaLaunchKernelEx(&config, token_logprobs_kernel<DTYPE, THREADS, SLOTS>, p), what);
}
// Threads for a row: as many as fill the GPU (148 x 1024), but no more than leave each a batch; above 512, which are several CTAs,
// as many as fill half of it, since clusters of CTAs are not placed as evenly.  us with 128 / 256 / 512 threads, and with 2 / 4 / 8
// CTAs of 512, without likeliest tokens and with 20:
//      1 x 50272 bf16     6.7  5.1  5.3   4.5  3.9  3.6          9.6  8.0  8.4    8.4  7.9  8.4
//     64 x 128257 bf16   14.1 10.3 10.0   7.5  7.6  9.8         21.4 13.8 13.1   11.6 12.2 22.9
//    200 x 50272 bf16     8.0  8.0  7.9                         12.8 11.2 11.5
//    600 x 50272 bf16    20.9 15.3 17.6                         27.1 20.6 26.4
//   2048 x 50272 bf16    38.3 40.8 54.6                         50.0 52.9 76.7
//   2048 x 50272 fp32    64.4 68.8 73.2                         76.4 80.4 91.7
//   2048 x 5000 bf16      8.5 12.0 22.4                         16.5 24.7 44.4
// 16-bit logits of CTAs of up to 256 threads travel through shared memory, where more of them fit than in registers (128 threads,
// without and with: 300 x 128257 27.7, 22.1; 2048 x 50272 43.7, 38.3; 2048 x 24000 22.8, 20.1; 2048 x 5000 8.5, 8.6).  Of 32 bits
// they gain nothing (2048 x 50272 63.7, 64.8), and with 512 threads there are seldom more than three batches.
// What bounds it: many rows of 16 bits the exponentials and instructions of a logit and HBM about equally (2048 x 50272 38 us,
// 5.4 TB/s), of 32 bits HBM (64 us, 6.45 TB/s); few rows a chain of waits (1 x 50272, 4 CTAs, 3.9 us, with 20 tokens 7.9).
struct Shape {
    int threads, parts;
};
Shape shape_for(int64_t rows, int64_t pieces) {
    int64_t threads = 128;
    while (threads < 512 * LP_MAX_PARTS && threads * 3 / 2 <= std::min<int64_t>((threads < 512 ? 151552 : 75776) / rows, pieces / 3)) threads *= 2;
    return {(int)std::min<int64_t>(threads, 512), (int)std::max<int64_t>(1, threads / 512)};
}
template <int DTYPE>
int launch(LogprobParams p, int64_t rows, cudaStream_t st, const char *what) {
    const Shape shape = shape_for(rows, ceil_div_i64(p.vocab, Logits<DTYPE>::PER));
    p.parts = shape.parts;
    return shape.threads == 128 ? launch_with<DTYPE, 128>(p, rows, st, what)
           : shape.threads == 256 ? launch_with<DTYPE, 256>(p, rows, st, what) : launch_with<DTYPE, 512>(p, rows, st, what);
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
    ATLAS_RETURN_IF((uintptr_t)q->logits % size || (uintptr_t)q->tokens % q->token_bytes || (((uintptr_t)q->logprobs | (uintptr_t)q->entropy) & 3) ||
                        (q->top && (((uintptr_t)q->top_logprobs & 3) || ((uintptr_t)q->top_tokens & 7))),
                    ATLAS_ERR_BAD_ARGUMENT, "%s: a buffer is not aligned to its type", what);
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
