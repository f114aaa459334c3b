// Attention of few queries over the 4-bit cache (decode, drafts).
//
// For the rows of one kv head (queries x query heads that share it) the cache is the 16-row operand of mma.m16n8k16 and the
// rows its 8 columns:
//   S[token][row] = sum over groups of 64 channels of s_token * sum (c - z) q       (c - z: exact small integers in fp16)
//   p = 2^(S' - m), O[channel][row] += sum over tokens of (s (c - z)) p             (s (c - z): exact in fp16)
// so that the only roundings are those of p to fp16 and of the output.  (s folded into p would save a product a pair, but p s
// in fp16 loses tokens whose scale is far below another's.)  A warp walks 16-token slabs, which it brings in by bulk copies of
// its own, with a softmax state of its own; nothing is shared until its range is done.
//
// Every (sequence, kv head) is a run of units (slabs that some row sees), and all runs together are cut evenly among the
// warps of one CTA per SM from the lengths on the device: ragged batches balance, and a captured graph serves any lengths.
// A run that lies within a warp goes straight to the output; pieces of the others are joined in shared memory, in order, and
// what goes beyond a CTA is left in the workspace for kv_join_kernel.
//
// Tokens that no row sees may hold anything: their scores are masked, and their values are zeros in the products.
//
// What bounds it: 2 x 131071 tokens of 8 kv heads, 302 MB, take 76 us (4.0 TB/s, 0.61 of the measured copy rate).  A slab of
// 128 channels (2304 bytes) costs 334 warp instructions, 250 of them its arithmetic (5 to extract, 4 to centre and, for
// values, 4 to scale 8 codes).  Issue slots are 60 % used and mma.sync holds the issue port for some 16 % more; in the
// rest all three warps of a scheduler wait for results of their own (few of them for DRAM).
// Two slabs at a time on 12 warps of 168 registers: brought in one by one they took 87 us, as one at a time on 16 warps of 128
// did, which is behind on short contexts (4001 tokens of 32 heads 22.5 us and 20.6); two at a time on 128 registers spills (129).
// (All four with masks in the pairs' code.)
// Short calls are a chain of waits: 1 us to plan, 1 to find pages, 1 for the first slab, 1 to join.
#include <algorithm>

#include "kv_attention.cuh"

namespace atlas {

namespace {

// A row tile of a sequence: its queries and the units that they see.
struct Run : Sequence {
    int sink_units, window_unit, units;   // units 0 .. sink_units - 1, then window_unit ...
    __device__ __forceinline__ int slab(int u) const { return u < sink_units ? u : u - sink_units + window_unit; }
};

__device__ __forceinline__ Run make_run(const Attention &a, int b, int row0, int rows) {
    Run r;
    static_cast<Sequence &>(r) = sequence(a, b);
    r.sink_units = r.window_unit = r.units = 0;
    const int64_t all = (int64_t)r.served(a) * a.group;
    if (row0 >= all) return r;
    const int p0 = r.start() + row0 / a.group, p1 = r.start() + (int)((min(all, (int64_t)row0 + rows) - 1) / a.group);
    if (p1 < 0) return r;
    const int end = p1 / KV_SLAB + 1;
    if (a.window) {
        r.window_unit = max(0, p0 - a.window + 1) / KV_SLAB;
        r.sink_units = min((min(a.sinks, p1 + 1) + KV_SLAB - 1) / KV_SLAB, r.window_unit);
    }
    r.units = r.sink_units + end - r.window_unit;
    return r;
}

// Units of all runs, and of those of the sequences in front of b: the same in every warp that asks.
__device__ __forceinline__ uint32_t count_units(const Attention &a, int row0, int rows, int b, uint32_t &in_front) {
    uint32_t sum = 0, front = 0;
    for (int k = threadIdx.x & 31; k < a.batch; k += 32) {
        const uint32_t units = make_run(a, k, row0, rows).units;
        sum += units;
        if (k < b) front += units;
    }
    in_front = __reduce_add_sync(0xffffffffu, front) * a.kv_heads;
    return __reduce_add_sync(0xffffffffu, sum) * a.kv_heads;
}
__device__ __forceinline__ uint32_t units_per_warp(uint32_t total, uint32_t warps) { return max((total + warps - 1) / warps, 1u); }

// Few short runs take a CTA each, and nothing is left to join: no more runs than CTAs, none longer than this.  (4 sequences of 900
// tokens on 32 kv heads of 128 channels 12.1 us and 15.3 cut evenly, 1 of 1000 on 8 12.0 and 11.6; on 8 of 256 channels 17.0 and
// 14.6, of 500 9.3 and 10.8.)
constexpr int kv_whole_units(int d) { return d == 256 ? 32 : 64; }
template <int D>
__device__ __forceinline__ bool whole_runs(const Attention &a, int row0, int rows) {
    if (!a.few_runs) return false;
    bool all = true;
    for (int k = threadIdx.x & 31; k < a.batch; k += 32) all = all && make_run(a, k, row0, rows).units <= kv_whole_units(D);
    return __all_sync(0xffffffffu, all);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// A lane's words of codes: 8 or 16 bytes, in each of two planes if D is 256.
template <int D>
__device__ __forceinline__ void read_words(const uint8_t *p, uint32_t (&w)[D / 32]) {
    if constexpr (D == 64) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + i * 1024);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}
template <int N>
__device__ __forceinline__ void read_params(const uint8_t *p, uint32_t (&w)[N]) {
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + i * 16);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}

template <int D, int NT, int WARPS, int STAGES>
struct Shape {
    static constexpr int ROWS = 8 * NT, GROUPS = D / 64, WORDS = D / 32;   // words: a lane's, of a token's key
    static constexpr int SLAB = kv_slab_bytes(D);
    static constexpr int PIECE_BYTES = D == 64 ? 8 : 16, KEY_ROW = 4 * PIECE_BYTES;   // of a lane's codes (in a plane); of a token's
    static constexpr int PIECE = ROWS * (D + 2) * 4;       // maximum, sum and output of the rows
    static constexpr int RING = STAGES * 2 * SLAB;         // a warp's pairs of slabs; holds its last piece in the end
    static constexpr int SMEM = WARPS * (RING + PIECE + STAGES * 8 + 2 * 16 + 32 * 8);
    static_assert(STAGES * WARPS % 2 == 0 && SMEM <= 227 * 1024, "shared memory");
    static_assert(PIECE <= RING, "a piece has to fit the ring");
};

// The state of a warp: maxima, sums and outputs of the rows in the layout of the accumulators.
template <int D, int NT>
struct State {
    float o[NT][D / 16][4];
    float l[NT][4];
    float m[NT][2];              // of rows 2 t and 2 t + 1, log2; -inf before the first visible score
    float ref[NT][2];            // what is taken from a score: m - 6, or 0 before the first
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[n][i][k] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) l[n][k] = 0.0f;
            m[n][0] = m[n][1] = -INFINITY;
            ref[n][0] = ref[n][1] = 0.0f;
        }
    }
};

// Four channels of a row of a piece (maxima, sums, outputs of its rows), brought to the maximum m of all pieces.
__device__ __forceinline__ void add_piece(const float *piece, int rows, int row, int d, int c, float m, float &l, float4 &o) {
    const float pm = piece[row], w = pm == -INFINITY ? 0.0f : exp2_fast(pm - m);
    const float4 po = *reinterpret_cast<const float4 *>(piece + 2 * rows + row * d + c);
    l = fmaf(piece[rows + row], w, l);
    o.x = fmaf(po.x, w, o.x), o.y = fmaf(po.y, w, o.y), o.z = fmaf(po.z, w, o.z), o.w = fmaf(po.w, w, o.w);
}
template <bool BF16>
__device__ __forceinline__ void store_row(char *dst, int c, float l, const float4 &o) {
    const float inv = l > 0.0f || l != l ? __frcp_rn(l) : 0.0f;
    if (dst) *reinterpret_cast<uint2 *>(dst + c * 2) = pack4<BF16>(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <int D, int NT, int WARPS, int STAGES, bool BF16>
__global__ void __launch_bounds__(WARPS * 32, 1) kv_attention_kernel(const Attention a) {
    using S = Shape<D, NT, WARPS, STAGES>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *const ring_all = smem, *const heads_all = smem + WARPS * S::RING;
    uint64_t *const bars = reinterpret_cast<uint64_t *>(heads_all + WARPS * S::PIECE);
    // of every warp's first and last piece: its run (sequence * kv_heads + head) or -1, 1 if the run ends there + 2 if it began
    // before, first query and queries of the sequence
    int4 *const notes = reinterpret_cast<int4 *>(bars + WARPS * STAGES);
    uint64_t *const slabs = reinterpret_cast<uint64_t *>(notes + 2 * WARPS) + (threadIdx.x / 32) * 32;

    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
    const int row0 = blockIdx.y * S::ROWS;
    const uint32_t ring = smem_u32(ring_all + warp * S::RING);
    const uint8_t *const ring_ptr = ring_all + warp * S::RING;
    const uint32_t bar = smem_u32(bars + warp * STAGES);
    if (lane < STAGES) mbar_init(bar + 8 * lane, 1);
    if (lane == 0) notes[2 * warp].x = notes[2 * warp + 1].x = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    wait_for_front();

    // Runs of the first 32 sequences, one a lane, and where they end among all units; those of more sequences are found again.
    auto ends_of = [&](const Run &r) {
        uint32_t sum = (uint32_t)r.units * a.kv_heads;
#pragma unroll
        for (int k = 1; k < 32; k *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, sum, k);
            if (lane >= k) sum += other;
        }
        return sum;
    };
    auto run_of = [&](int b) {
        Run r = {};
        if (b < a.batch) r = make_run(a, b, row0, S::ROWS);
        return r;
    };
    Run mine = run_of(lane), run = {};
    int b = 0, head = 0, unit = 0, todo = 0;
    if (whole_runs<D>(a, row0, S::ROWS)) {
        b = blockIdx.x / a.kv_heads, head = blockIdx.x - b * a.kv_heads;
        run = run_of(b);
        const int share = (run.units + WARPS - 1) / WARPS;
        unit = warp * share;
        todo = min(run.units, unit + share) - unit;
        if (run.units == 0 && b < a.batch)
            for (int x = threadIdx.x; x < S::ROWS * (D / 4); x += WARPS * 32)
                store_row<BF16>(out_row(a, run, head, row0 + x / (D / 4), D), x % (D / 4) * 4, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    } else {
        uint32_t ends = ends_of(mine);
        uint32_t total = __shfl_sync(0xffffffffu, ends, 31);
        for (int base = 32; base < a.batch; base += 32) total += __reduce_add_sync(0xffffffffu, (uint32_t)run_of(base + lane).units) * a.kv_heads;
        const uint32_t quota = units_per_warp(total, gridDim.x * WARPS);
        const uint32_t begin = (blockIdx.x * WARPS + warp) * quota, end = min(total, begin + quota);
        if (begin < end) {
            // the sequence, head and unit that the range begins with
            uint32_t before = 0, past;
            int base = 0;
            while (!(past = __ballot_sync(0xffffffffu, before + ends > begin))) {
                before += __shfl_sync(0xffffffffu, ends, 31);
                base += 32;
                mine = run_of(base + lane);
                ends = ends_of(mine);
            }
            const int at_lane = __ffs(past) - 1;
            b = base + at_lane;
            run.first_query = __shfl_sync(0xffffffffu, mine.first_query, at_lane);
            run.length = __shfl_sync(0xffffffffu, mine.length, at_lane);
            run.queries = __shfl_sync(0xffffffffu, mine.queries, at_lane);
            run.sink_units = __shfl_sync(0xffffffffu, mine.sink_units, at_lane);
            run.window_unit = __shfl_sync(0xffffffffu, mine.window_unit, at_lane);
            run.units = __shfl_sync(0xffffffffu, mine.units, at_lane);
            const uint32_t in_sequence = begin - (before + __shfl_sync(0xffffffffu, ends, at_lane) - (uint32_t)run.units * a.kv_heads);
            head = (int)(in_sequence / (uint32_t)run.units);
            unit = (int)(in_sequence - (uint32_t)head * run.units);
            todo = (int)(end - begin);
        }
    }

    if (todo > 0) {
        // The producer's own place, up to STAGES pairs of units ahead (a run's last may be one).  Every lane finds the slab of one of the next 32 units of its run
        // (0: not in the cache); lane 0 asks for them one by one.
        Run p_run = run;
        int p_b = b, p_head = head, p_unit = unit, p_left = 0, issued = 0, asked = 0, p_stage = 0;
        uint32_t absent = 0;   // of each stage two bits: slabs that are not in the cache (they are passed over)
        const uint64_t *p_next = slabs;
        auto produce = [&]() {
            if (issued >= todo) return;
            if (p_left == 0) {
                if (p_unit >= p_run.units) {
                    p_unit = 0;
                    if (++p_head == a.kv_heads) {
                        p_head = 0;
                        do p_run = make_run(a, ++p_b, row0, S::ROWS); while (p_run.units == 0);
                    }
                }
                p_left = min(32, p_run.units - p_unit);
                __syncwarp();    // (lane 0 has read the last 32)
                if (lane < p_left) {
                    const int token = p_run.slab(p_unit + lane) * KV_SLAB, in_table = token / a.page_size;
                    const int page = a.page_table[p_b * a.table_stride + in_table];
                    const uint8_t *src = a.cache + (((int64_t)page * a.kv_heads + p_head) * (a.page_size / KV_SLAB) + (token - in_table * a.page_size) / KV_SLAB) * S::SLAB;
                    slabs[lane] = page >= 0 && page < a.num_pages ? reinterpret_cast<uint64_t>(src) : 0;
                }
                __syncwarp();
                p_unit += p_left;
                p_next = slabs;
            }
            const int count = min(min(2, p_left), todo - issued);
            const uint64_t src0 = p_next[0], src1 = count == 2 ? p_next[1] : 0;
            absent = (absent & ~(3u << (2 * p_stage))) | ((src0 ? 0u : 1u) | (src1 ? 0u : 2u)) << (2 * p_stage);
            if (lane == 0) {
                const uint32_t at = bar + 8 * p_stage, dst = ring + p_stage * (2 * S::SLAB);
                mbar_arrive_expect_tx(at, (src0 ? S::SLAB : 0) + (src1 ? S::SLAB : 0));
                if (src0 && src1 == src0 + S::SLAB) {
                    bulk_load_1d(dst, reinterpret_cast<const void *>(src0), 2 * S::SLAB, at);
                } else {
                    if (src0) bulk_load_1d(dst, reinterpret_cast<const void *>(src0), S::SLAB, at);
                    if (src1) bulk_load_1d(dst + S::SLAB, reinterpret_cast<const void *>(src1), S::SLAB, at);
                }
            }
            p_next += count;
            p_left -= count;
            issued += count;
            ++asked;
            p_stage = p_stage + 1 == STAGES ? 0 : p_stage + 1;
        };
        for (int i = 0; i < STAGES; ++i) produce();

        State<D, NT> st;
        uint32_t qf[NT][S::WORDS][4];
        float factor[NT][2];       // log2 units of a row's scores
        int place[NT][2];          // positions of rows 2 t and 2 t + 1, -1: no such row
        int plain_sinks = 0, plain_from = 0, plain_count = 0;   // slabs that all rows see whole: below the first, and so many from the second on
        int seen_from = 0;         // first token in the window of any row
        auto plain = [&](int slab) { return slab < plain_sinks || (uint32_t)(slab - plain_from) < (uint32_t)plain_count; };
        bool fresh = true, first_piece = true, failed = false;
        const bool begins_inside = unit != 0;
        int done = 0, taken = 0, stage = 0;
        uint32_t parity = 0;

        auto leave = [&](bool whole_run, bool ends_here) {
            // to the output (a run that began and ended here), or to shared memory
            if (whole_run) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        char *dst = out_row(a, run, head, row0 + 8 * n + 2 * t + e, D);
                        const float inv = st.l[n][e] > 0.0f || st.l[n][e] != st.l[n][e] ? 1.0f / st.l[n][e] : 0.0f;
#pragma unroll
                        for (int j = 0; j < S::WORDS; ++j)
                            if (dst)
                                *reinterpret_cast<uint2 *>(dst + (32 * j + 4 * g) * 2) =
                                    pack4<BF16>(st.o[n][2 * j][e] * inv, st.o[n][2 * j][2 + e] * inv, st.o[n][2 * j + 1][e] * inv, st.o[n][2 * j + 1][2 + e] * inv);
                    }
                return;
            }
            float *piece = reinterpret_cast<float *>(first_piece ? heads_all + warp * S::PIECE : ring_all + warp * S::RING);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 8 * n + 2 * t + e;
                    if (g == 0) {
                        piece[row] = st.m[n][e];
                        piece[S::ROWS + row] = st.l[n][e];
                    }
#pragma unroll
                    for (int j = 0; j < S::WORDS; ++j)
                        *reinterpret_cast<float4 *>(piece + 2 * S::ROWS + row * D + 32 * j + 4 * g) =
                            make_float4(st.o[n][2 * j][e], st.o[n][2 * j][2 + e], st.o[n][2 * j + 1][e], st.o[n][2 * j + 1][2 + e]);
                }
            if (lane == 0) notes[2 * warp + (first_piece ? 0 : 1)] = make_int4(b * a.kv_heads + head, (ends_here ? 1 : 0) + (first_piece && begins_inside ? 2 : 0), run.first_query, run.queries);
        };

        // Two slabs of the run that all rows see whole (their chains of products and exponentials overlap), or any one.  (With masks
        // in the pair's code 2 x 131071 tokens take 79 us instead of 76, with a third form of it 78.)
        auto work = [&](auto count, const uint8_t *const (&slab)[2], const int (&at)[2]) {
            constexpr int N = decltype(count)::value;
            float s[N][NT][4];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                uint32_t low[S::WORDS], high[S::WORDS], kl[S::GROUPS], kh[S::GROUPS];
                read_words<D>(slab[u] + g * S::KEY_ROW + t * S::PIECE_BYTES, low);
                read_words<D>(slab[u] + (g + 8) * S::KEY_ROW + t * S::PIECE_BYTES, high);
                read_params<S::GROUPS>(slab[u] + kv_key_params(D) + g * S::GROUPS * 4, kl);
                read_params<S::GROUPS>(slab[u] + kv_key_params(D) + (g + 8) * S::GROUPS * 4, kh);
#pragma unroll
                for (int gr = 0; gr < S::GROUPS; ++gr) {
                    const __half2 lo = h2(kl[gr]), hi = h2(kh[gr]);
                    const __half2 bl = __high2half2(lo), bh = __high2half2(hi), bl16 = minus16_of(bl), bh16 = minus16_of(bh);
                    float acc[NT][4];
#pragma unroll
                    for (int j = 2 * gr; j < 2 * gr + 2; ++j) {
                        __half2 x[4], y[4];
                        open_word(low[j], bl, bl16, x);
                        open_word(high[j], bh, bh16, y);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                if (j == 2 * gr && i == 0)
                                    mma_f16_new(acc[n], h2(x[2 * i]), h2(y[2 * i]), h2(x[2 * i + 1]), h2(y[2 * i + 1]), qf[n][j][2 * i], qf[n][j][2 * i + 1]);
                                else
                                    mma_f16(acc[n], h2(x[2 * i]), h2(y[2 * i]), h2(x[2 * i + 1]), h2(y[2 * i + 1]), qf[n][j][2 * i], qf[n][j][2 * i + 1]);
                            }
                    }
                    const float sl = __low2float(lo), sh = __low2float(hi);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) s[u][n][k] = gr ? fmaf(acc[n][k], k < 2 ? sl : sh, s[u][n][k]) : acc[n][k] * (k < 2 ? sl : sh);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[u][n][k] *= factor[n][k & 1];
                if (N == 1 && !plain(at[u])) {
                    const int token0 = at[u] * KV_SLAB;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int token = token0 + g + (k / 2) * 8, p = place[n][k & 1];
                            if (token > p || (a.window && token <= p - a.window && token >= a.sinks)) s[u][n][k] = -INFINITY;
                        }
                }
            }
            // the maximum moves only where a score passes it by more than 2^8
            float tops[NT][2];
            bool passes = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    tops[n][e] = fmaxf(s[0][n][e], s[0][n][2 + e]);
                    if (N == 2) tops[n][e] = fmaxf(tops[n][e], fmaxf(s[N - 1][n][e], s[N - 1][n][2 + e]));
                    passes |= tops[n][e] > st.m[n][e] + KV_HEADROOM;
                }
            if (__any_sync(0xffffffffu, passes)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(tops[n][e], st.m[n][e]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float shrink = st.m[n][e] == -INFINITY ? 0.0f : exp2_fast(st.m[n][e] - top);
                        st.m[n][e] = top;
                        st.ref[n][e] = top == -INFINITY ? 0.0f : top - KV_SHIFT;
                        st.l[n][e] *= shrink, st.l[n][2 + e] *= shrink;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) st.o[n][i][e] *= shrink, st.o[n][i][2 + e] *= shrink;
                    }
            }
            uint32_t pb[N][NT][2];
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float p[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) p[k] = exp2_fast(s[u][n][k] - st.ref[n][k & 1]);
                    pb[u][n][0] = transpose8x8(h2(__floats2half2_rn(p[0], p[1])));
                    pb[u][n][1] = transpose8x8(h2(__floats2half2_rn(p[2], p[3])));
                }
#pragma unroll
            for (int u = 0; u < N; ++u) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    mma_f16(st.l[n], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[u][n][0], pb[u][n][1]);   // sums of what is used
                // outputs
                uint32_t v0[S::WORDS], v1[S::WORDS], q0[2 * S::GROUPS], q1[2 * S::GROUPS];
                read_words<D>(slab[u] + kv_value_codes(D) + lane * S::PIECE_BYTES, v0);
                read_words<D>(slab[u] + kv_value_codes(D) + 32 * S::PIECE_BYTES + lane * S::PIECE_BYTES, v1);
                read_params<2 * S::GROUPS>(slab[u] + kv_value_params(D) + t * S::GROUPS * 8, q0);
                read_params<2 * S::GROUPS>(slab[u] + kv_value_params(D) + (t + 4) * S::GROUPS * 8, q1);
                if (N == 1 && !plain(at[u])) {   // tokens that no row sees may hold anything: zeros (their weights are zero too, but not times NaN)
                    const int token = at[u] * KV_SLAB + 2 * t;
                    auto seen = [&](int k) { return k < run.length && (k >= seen_from || k < a.sinks); };
                    const uint32_t keep0 = (seen(token) ? 0xffffu : 0u) | (seen(token + 1) ? 0xffff0000u : 0u);
                    const uint32_t keep1 = (seen(token + 8) ? 0xffffu : 0u) | (seen(token + 9) ? 0xffff0000u : 0u);
#pragma unroll
                    for (int gr = 0; gr < S::GROUPS; ++gr) {
                        q0[2 * gr] &= keep0, q0[2 * gr + 1] = (q0[2 * gr + 1] & keep0) | (0x64006400u & ~keep0);
                        q1[2 * gr] &= keep1, q1[2 * gr + 1] = (q1[2 * gr + 1] & keep1) | (0x64006400u & ~keep1);
                    }
                }
#pragma unroll
                for (int gr = 0; gr < S::GROUPS; ++gr) {
                    const __half2 s0 = h2(q0[2 * gr]), s1 = h2(q1[2 * gr]), b0 = h2(q0[2 * gr + 1]), b1 = h2(q1[2 * gr + 1]);
                    const __half2 b016 = minus16_of(b0), b116 = minus16_of(b1);
#pragma unroll
                    for (int j = 2 * gr; j < 2 * gr + 2; ++j) {
                        __half2 x[4], y[4];
                        open_word(v0[j], b0, b016, x);
                        open_word(v1[j], b1, b116, y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = __hmul2(x[i], s0), y[i] = __hmul2(y[i], s1);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
                                mma_f16(st.o[n][2 * j + i], h2(x[2 * i]), h2(x[2 * i + 1]), h2(y[2 * i]), h2(y[2 * i + 1]), pb[u][n][0], pb[u][n][1]);
                    }
                }
            }
        };

        while (done < todo) {
            if (fresh) {           // another run: its queries into registers
                st.clear();
                fresh = false;
                const int past = max(0, run.start() + row0 / a.group + 1);   // of the tokens that the first row may see
                seen_from = a.window ? max(0, past - a.window) : 0;
                plain_from = a.window ? max(0, run.length - 1 - a.window + KV_SLAB) / KV_SLAB : 0;
                plain_count = max(0, past / KV_SLAB - plain_from);
                plain_sinks = min(a.sinks, past) / KV_SLAB;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int row = row0 + 8 * n + g, query = row / a.group;
                    const bool there = query < run.served(a);
                    const char *src = a.q + (int64_t)(run.first_query + query) * a.q_token_stride + (head * a.group + row % a.group) * a.q_head_stride;
                    float top = 0.0f;
                    uint4 raw[S::WORDS];
#pragma unroll
                    for (int j = 0; j < S::WORDS; ++j) {
                        raw[j] = there ? *reinterpret_cast<const uint4 *>(src + (32 * j + 8 * t) * 2) : make_uint4(0, 0, 0, 0);
                        if (BF16) {
                            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
                        }
                    }
                    float unscale = 1.0f;
                    if (BF16) {
                        // bf16 rows become fp16 times a power of two, chosen so that the largest is in [1, 2): exact, but for
                        // numbers below 2^-14 of it, which are off by 2^-25 of it at most
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        const int ex = min(max((__float_as_int(top) >> 23) & 0xff, 8), 246);
                        const float down = __int_as_float((254 - ex) << 23);
                        unscale = __int_as_float(ex << 23);
#pragma unroll
                        for (int j = 0; j < S::WORDS; ++j) {
                            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                qf[n][j][i] = h2(__floats2half2_rn(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i] & 0xffff0000u) * down));
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < S::WORDS; ++j) qf[n][j][0] = raw[j].x, qf[n][j][1] = raw[j].y, qf[n][j][2] = raw[j].z, qf[n][j][3] = raw[j].w;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        factor[n][e] = a.scale_log2 * __shfl_sync(0xffffffffu, unscale, (2 * t + e) * 4);
                        const int r = row0 + 8 * n + 2 * t + e;
                        place[n][e] = r / a.group < run.served(a) ? run.start() + r / a.group : -1;
                    }
                }
            }

            if (!__all_sync(0xffffffffu, mbar_try_wait(bar + 8 * stage, parity)) && !__all_sync(0xffffffffu, mbar_wait(bar + 8 * stage, parity))) {
                failed = true;
                break;
            }
            const int two = min(min(2, run.units - unit), todo - done);
            const uint8_t *slab[2] = {ring_ptr + stage * (2 * S::SLAB), ring_ptr + stage * (2 * S::SLAB) + S::SLAB};
            const int at[2] = {run.slab(unit), run.slab(unit + 1)};
            const bool there[2] = {!(absent >> (2 * stage) & 1), !(absent >> (2 * stage) & 2)};   // (of the second: if there are two)
            ++taken;
            if (++stage == STAGES) stage = 0, parity ^= 1;
            if (two == 2 && there[0] && there[1] && plain(at[0]) && plain(at[1])) {
                work(std::integral_constant<int, 2>(), slab, at);
            } else {
#pragma unroll 1
                for (int u = 0; u < two; ++u) {
                    const uint8_t *const one_slab[2] = {u ? slab[1] : slab[0], nullptr};
                    const int one_at[2] = {u ? at[1] : at[0], 0};
                    if (u ? there[1] : there[0]) work(std::integral_constant<int, 1>(), one_slab, one_at);
                }
            }
            __syncwarp();          // everyone has read the stages
            produce();
            done += two;
            unit += two;

            if (unit == run.units) {
                const bool whole = !(first_piece && begins_inside);
                leave(whole, true);
                first_piece = false;
                fresh = true;
                unit = 0;
                if (done < todo && ++head == a.kv_heads) {
                    head = 0;
                    do run = make_run(a, ++b, row0, S::ROWS); while (run.units == 0);
                }
            }
        }
        if (failed) {              // a copy that never came: those in flight land (or not, within the limit) before the CTA goes
            for (int i = taken; i < asked; ++i) mbar_wait(bar + 8 * (i % STAGES), (i / STAGES) & 1);
            if (lane == 0 && a.status) *a.status = 1;
        } else if (unit) {
            __syncwarp();
            leave(false, false);
        }
    }
    __syncthreads();

    // Pieces in order: runs that are whole within the CTA go to the output, the others to the workspace.  Lane k looks at note k.
    static_assert(2 * WARPS <= 32, "a lane a note");
    const int4 note = lane < 2 * WARPS ? notes[lane] : make_int4(-1, 0, 0, 0);
    for (uint32_t left = __ballot_sync(0xffffffffu, note.x >= 0); left;) {
        const int i = __ffs(left) - 1, id = __shfl_sync(0xffffffffu, note.x, i);
        const uint32_t members = __ballot_sync(0xffffffffu, note.x == id);
        left &= ~members;
        const bool ends_here = __any_sync(0xffffffffu, note.x == id && (note.y & 1));
        const bool begins_here = !(i == 0 && (__shfl_sync(0xffffffffu, note.y, 0) & 2));   // (only the CTA's first piece can have begun before it)
        Sequence seq;
        seq.first_query = __shfl_sync(0xffffffffu, note.z, i), seq.queries = __shfl_sync(0xffffffffu, note.w, i);
        const int head = id % a.kv_heads, w0 = i / 2, w1 = (31 - __clz(members)) / 2;
        for (int x = threadIdx.x; x < S::ROWS * (D / 4); x += WARPS * 32) {
            const int row = x / (D / 4), c = x % (D / 4) * 4;
            // first pieces are a piece apart, last ones a ring
            float m = -INFINITY;
#pragma unroll 4
            for (int w = w0; w <= w1; ++w) {
                if (members >> (2 * w) & 1) m = fmaxf(m, reinterpret_cast<const float *>(heads_all + w * S::PIECE)[row]);
                if (members >> (2 * w) & 2) m = fmaxf(m, reinterpret_cast<const float *>(ring_all + w * S::RING)[row]);
            }
            float l = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int w = w0; w <= w1; ++w) {
                if (members >> (2 * w) & 1) add_piece(reinterpret_cast<const float *>(heads_all + w * S::PIECE), S::ROWS, row, D, c, m, l, o);
                if (members >> (2 * w) & 2) add_piece(reinterpret_cast<const float *>(ring_all + w * S::RING), S::ROWS, row, D, c, m, l, o);
            }
            if (begins_here && ends_here) {
                store_row<BF16>(out_row(a, seq, head, row0 + row, D), c, l, o);
            } else {
                float *piece = a.partial + (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + (begins_here ? 1 : 0)) * (S::PIECE / 4);
                if (c == 0) piece[row] = m, piece[S::ROWS + row] = l;
                *reinterpret_cast<float4 *>(piece + 2 * S::ROWS + row * D + c) = o;
            }
        }
    }
}

// One CTA a run: joins what several CTAs of kv_attention_kernel have left of it, in their order, and zeroes rows of runs
// without units and rows that are no sequence's.  It finds the CTAs from the lengths, before the kernel in front has ended (which began when they were there).
template <int D, int NT, int WARPS, bool BF16>
__global__ void __launch_bounds__(256) kv_join_kernel(const Attention a, int ctas) {
    constexpr int ROWS = 8 * NT, PIECE = ROWS * (D + 2);
    const int b = blockIdx.x / a.kv_heads, head = blockIdx.x - b * a.kv_heads, row0 = blockIdx.y * ROWS;
    const Run run = make_run(a, b, row0, ROWS);
    uint32_t first;
    const uint32_t quota = units_per_warp(count_units(a, row0, ROWS, b, first), (uint32_t)ctas * WARPS) * WARPS;
    const bool whole = whole_runs<D>(a, row0, ROWS);
    first += (uint32_t)head * run.units;
    const int c0 = first / quota, c1 = run.units ? (first + run.units - 1) / quota : c0;
    if (blockIdx.y == 0) zero_rows_next_to(a, run, b, D, head * 256 + threadIdx.x, (int64_t)a.kv_heads * 256);
    // (CTAs without work wait too: what follows this kernel takes its end for that of the kernel in front)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (whole || (run.units && c0 == c1)) return;
    for (int x = threadIdx.x; x < ROWS * (D / 4); x += 256) {
        const int row = x / (D / 4), c = x % (D / 4) * 4;
        char *dst = out_row(a, run, head, row0 + row, D);
        if (!dst) continue;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k0 = run.units ? c0 : c1 + 1; k0 <= c1; k0 += 4) {   // four pieces' loads at a time
            float pm[4], pl[4];
            float4 po[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = min(k0 + u, c1);
                const float *piece = a.partial + (((int64_t)blockIdx.y * ctas + k) * 2 + (k == c0 ? 1 : 0)) * PIECE;
                pm[u] = k0 + u <= c1 ? piece[row] : -INFINITY;
                pl[u] = piece[ROWS + row];
                po[u] = *reinterpret_cast<const float4 *>(piece + 2 * ROWS + row * D + c);
            }
            const float top = fmaxf(m, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])));
            const float keep = m == -INFINITY ? 0.0f : exp2_fast(m - top);
            m = top;
            l *= keep, o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float w = pm[u] == -INFINITY ? 0.0f : exp2_fast(pm[u] - top);
                if (k0 + u > c1) break;
                l = fmaf(pl[u], w, l);
                o.x = fmaf(po[u].x, w, o.x), o.y = fmaf(po[u].y, w, o.y), o.z = fmaf(po[u].z, w, o.z), o.w = fmaf(po[u].w, w, o.w);
            }
        }
        store_row<BF16>(dst, c, l, o);
    }
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    static thread_local int known_dev = -1, known = 0;
    if (known_dev != dev) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
        known_dev = dev, known = sms;
    }
    return known;
}

struct Plan {
    int nt, warps, stages;
    int64_t tiles;
    size_t piece_bytes;
};
Plan plan_of(const AtlasKvAttention &p) {
    Plan plan;
    const int64_t rows = p.max_queries * (p.q_heads / p.kv_heads);
    // Rows 8 at a time, or 16, which takes 1.7 times as long a slab and more to start and to join: for 9 to 16 and 25 to 32 rows
    // of 128 channels and contexts that may be long (16 sequences of 8000 tokens, 16 rows: 49 us 8 at a time, 42 16 at a time;
    // 4 of 4000 on 2 kv heads: 15 and 24; 8 of 4000, 24 rows: 40 and 41).
    const int64_t slabs = p.batch * p.kv_heads * (p.max_pages * p.page_size / KV_SLAB);
    plan.nt = p.head_dim == 128 && ceil_div_i64(rows, 8) % 2 == 0 && slabs >= 12000 ? 2 : 1;
    plan.tiles = ceil_div_i64(std::max<int64_t>(rows, 1), 8 * plan.nt);
    plan.piece_bytes = (size_t)8 * plan.nt * (p.head_dim + 2) * 4;
    return plan;
}

template <int D, int NT, int WARPS, int STAGES, bool BF16>
int launch(const Attention &a, int64_t tiles, int ctas, cudaStream_t stream) {
    using S = Shape<D, NT, WARPS, STAGES>;
    const char *what = "atlas_kv_attention";
    auto *kernel = kv_attention_kernel<D, NT, WARPS, STAGES, BF16>;
    int e = allow_smem<kv_attention_kernel<D, NT, WARPS, STAGES, BF16>>(S::SMEM, what);
    if (e == ATLAS_OK) e = launch_early(kernel, dim3((unsigned)ctas, (unsigned)tiles), WARPS * 32, S::SMEM, stream, what, a);
    if (e != ATLAS_OK || (a.few_runs && a.max_tokens <= kv_whole_units(D) * KV_SLAB && !a.query_starts)) return e;
    return launch_early(kv_join_kernel<D, NT, WARPS, BF16>, dim3((unsigned)(a.batch * a.kv_heads), (unsigned)tiles), 256, 0, stream, what, a, ctas);
}

template <int D, bool BF16>
int launch_nt(const Attention &a, const Plan &plan, int ctas, cudaStream_t stream) {
    // Warps and slabs in flight: what registers (168, 255) and shared memory hold.
    if constexpr (D == 64) return launch<64, 1, 12, 4, BF16>(a, plan.tiles, ctas, stream);
    if constexpr (D == 128) return plan.nt == 1 ? launch<128, 1, 12, 2, BF16>(a, plan.tiles, ctas, stream) : launch<128, 2, 8, 3, BF16>(a, plan.tiles, ctas, stream);
    if constexpr (D == 256) return launch<256, 1, 8, 2, BF16>(a, plan.tiles, ctas, stream);
    return ATLAS_ERR_UNSUPPORTED;
}

bool aligned16(const void *p, int64_t a, int64_t b) { return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)a | (uintptr_t)b) & 15); }

int check_arguments(const AtlasKvAttention *p, const char *what) {
    ATLAS_RETURN_IF(!p, ATLAS_ERR_BAD_ARGUMENT, "%s: no arguments", what);
    const int shape = check_kv_shape(p->num_pages, p->kv_heads, p->head_dim, p->page_size, what);
    if (shape != ATLAS_OK) return shape;
    ATLAS_RETURN_IF(p->dtype != ATLAS_DTYPE_F16 && p->dtype != ATLAS_DTYPE_BF16, ATLAS_ERR_BAD_ARGUMENT, "%s: dtype %d", what, p->dtype);
    ATLAS_RETURN_IF(p->q_heads < 1 || p->q_heads % p->kv_heads || p->q_heads / p->kv_heads > 1024, ATLAS_ERR_BAD_ARGUMENT,
                    "%s: %d query heads on %d kv heads", what, p->q_heads, p->kv_heads);
    ATLAS_RETURN_IF(p->total_queries < 0 || p->batch < 0 || p->max_queries < 0 || p->window < 0 || p->sinks < 0 || p->max_pages < 0,
                    ATLAS_ERR_BAD_ARGUMENT, "%s: negative size", what);
    ATLAS_RETURN_IF(p->total_queries > (1 << 24) || p->batch * (int64_t)p->kv_heads > 0x7fffffff || p->max_queries > (1 << 24) ||
                        p->max_pages * (int64_t)p->page_size > (1 << 30) || p->batch * (int64_t)p->kv_heads * (p->max_pages * (int64_t)p->page_size / KV_SLAB + 1) > 0x7fffffff,
                    ATLAS_ERR_UNSUPPORTED, "%s: %lld queries of %lld sequences over up to %lld tokens", what, (long long)p->total_queries,
                    (long long)p->batch, (long long)p->max_pages * p->page_size);
    return ATLAS_OK;
}

}  // namespace
}  // namespace atlas

extern "C" {

size_t atlas_kv_attention_workspace_bytes(const AtlasKvAttention *p) {
    using namespace atlas;
    if (check_arguments(p, "atlas_kv_attention_workspace_bytes") != ATLAS_OK) return 0;
    if (kv_prompt_serves(*p)) return kv_prompt_workspace_bytes(*p);
    const Plan plan = plan_of(*p);
    return (size_t)plan.tiles * std::max<int64_t>(1, sm_count() / plan.tiles) * 2 * plan.piece_bytes;
}

int atlas_kv_attention(const AtlasKvAttention *p, void *stream) {
    using namespace atlas;
    clear_error();
    const char *what = "atlas_kv_attention";
    const int args = check_arguments(p, what);
    if (args != ATLAS_OK) return args;
    if (p->total_queries == 0 || (p->batch == 0 && !p->out)) return ATLAS_OK;
    if (p->batch == 0)   // (no sequence has them)
        return check_cuda(cudaMemsetAsync(p->out, 0, (size_t)p->total_queries * p->q_heads * p->head_dim * 2, (cudaStream_t)stream), what);
    ATLAS_RETURN_IF(!p->query_starts && p->total_queries % p->batch, ATLAS_ERR_BAD_ARGUMENT, "%s: %lld queries of %lld sequences without query_starts", what,
                    (long long)p->total_queries, (long long)p->batch);
    ATLAS_RETURN_IF(p->max_queries < (p->query_starts ? 1 : p->total_queries / p->batch), ATLAS_ERR_BAD_ARGUMENT, "%s: max_queries %lld", what,
                    (long long)p->max_queries);
    ATLAS_RETURN_IF(!p->q || !p->out || !p->lengths || (p->num_pages && !p->cache) || (p->max_pages && !p->page_table), ATLAS_ERR_BAD_ARGUMENT,
                    "%s: null pointer", what);
    const Plan plan = plan_of(*p);
    ATLAS_RETURN_IF((kv_prompt_serves(*p) ? kv_prompt_blocks(*p) : plan.tiles) > 65535, ATLAS_ERR_UNSUPPORTED, "%s: %lld queries in a sequence", what,
                    (long long)p->max_queries);
    ATLAS_RETURN_IF(!aligned16(p->q, 2 * p->q_token_stride, 2 * p->q_head_stride) || !aligned16(p->out, 0, 0) || !aligned16(p->cache, 0, 0) ||
                        (reinterpret_cast<uintptr_t>(p->workspace) & 255),
                    ATLAS_ERR_BAD_ARGUMENT, "%s: pointers and strides must be multiples of 16 bytes, the workspace of 256", what);
    const int dev = check_device();
    if (dev != ATLAS_OK) return dev;
    const int ctas = (int)std::max<int64_t>(1, sm_count() / plan.tiles);   // (all row tiles at a time)
    const size_t bytes = atlas_kv_attention_workspace_bytes(p);
    ATLAS_RETURN_IF(bytes && (!p->workspace || p->workspace_bytes < bytes), ATLAS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", what,
                    p->workspace_bytes, bytes);

    Attention a = {};
    a.q = (const char *)p->q, a.q_token_stride = 2 * p->q_token_stride, a.q_head_stride = 2 * p->q_head_stride;
    a.out = (char *)p->out, a.cache = (const uint8_t *)p->cache;
    a.page_table = p->page_table, a.lengths = p->lengths, a.query_starts = p->query_starts;
    a.partial = (float *)p->workspace, a.status = p->status;
    a.num_pages = p->num_pages, a.table_stride = p->table_stride, a.max_tokens = p->max_pages * p->page_size;
    a.total_queries = p->total_queries, a.uniform = p->query_starts ? 0 : p->total_queries / p->batch;
    a.max_queries = (int)p->max_queries;
    a.batch = (int)p->batch, a.q_heads = p->q_heads, a.kv_heads = p->kv_heads, a.group = p->q_heads / p->kv_heads;
    // A window of all tokens hides none: as no window it needs no masks, and position - window stays within 32 bits below (a query
    // may be at a negative position, and 2^31 - 1 is a usual "no window").
    a.page_size = p->page_size, a.window = p->window < a.max_tokens ? p->window : 0, a.sinks = p->sinks;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.few_runs = p->batch * p->kv_heads <= ctas;
    const bool bf16 = p->dtype == ATLAS_DTYPE_BF16;
    cudaStream_t s = (cudaStream_t)stream;
    if (kv_prompt_serves(*p)) return kv_prompt(a, *p, s);
    switch (p->head_dim) {
        case 64: return bf16 ? launch_nt<64, true>(a, plan, ctas, s) : launch_nt<64, false>(a, plan, ctas, s);
        case 128: return bf16 ? launch_nt<128, true>(a, plan, ctas, s) : launch_nt<128, false>(a, plan, ctas, s);
        default: return bf16 ? launch_nt<256, true>(a, plan, ctas, s) : launch_nt<256, false>(a, plan, ctas, s);
    }
}

}  // extern "C"
