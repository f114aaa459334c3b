// Attention of many queries over the 4-bit cache (prompts, chunks of prompts, long drafts) on the tensor cores.
//
// A CTA takes one kv head and two tiles of 128 rows (queries x the query heads that share the kv head; one tile if D is 256)
// and walks the tiles of 128 tokens (64) that any of them sees:
//   S = Q K^T      tcgen05, 128 rows x 128 tokens, both operands in shared memory (Q as fp16, bf16 rows times a power of two)
//   P = 2^(S' - m) a thread a row; P goes back to tensor memory as fp16, over S
//   O += P V       tcgen05, P from tensor memory, N = D channels, fp32 accumulators in tensor memory
// K and V are rebuilt from their codes into 128-byte-swizzled K-major tiles in shared memory, as the exact fp16 numbers that
// the cache stands for, so the only roundings are those of P and of the output.  (The sum of a row is that of its weights before
// they are rounded: values that are all alike can come out 2^-11 off.  Sums of the rounded ones, by adds of fp16 to fp32, took
// 176 us for 166.)  Tokens that no row sees may hold anything, as in kv_attention.cu.  The running maximum of a row follows its
// scores only where they pass it by 2^8 (O is rescaled then, which is rare); P keeps 14 bits of headroom for that.
//
// Warps: four of softmax for each row tile, three that rebuild keys and three that rebuild values, one that issues the MMAs,
// one that brings halves of slabs (keys, values) in by bulk copies, each half as far ahead as its ring has room.  While the
// softmax warps of one row tile work, the tensor core works on the other.
//
// What bounds it (4096 queries on 32 heads of 128 over 8 kv heads: 166 us by itself, 830 TFLOP/s, half of the measured peak; 170
// to 175 us in passes through the entry point, by the power that is left): a CTA needs
// 2800 cycles for a tile of 128 tokens, of which the tensor core works 2048 at its peak rate, and some 23000 for its start and end
// (14000 until the first S: rows of Q by bulk copies, slabs, rebuilding; 7000 behind the last P), a fifth of the largest.  In
// the loop the chain of a row tile (S, maximum, weights, P, two products) is the bound: exponentials replaced by copies gave 7 %,
// a polynomial for a quarter of them 0 %.  Built and slower: S in two buffers of 64 tokens for each row tile (an MMA of 64
// columns with both operands in shared memory takes 80 cycles, one of 128 91; 5300 cycles for 128 tokens), two threads a row
// (178 us against 173 then), registers shared out unevenly (setmaxnreg: spills), one pass over S that keeps P in registers
// until the maximum is known (code too long for the instruction cache; 5400 cycles).
#include <algorithm>

#include "kv_attention.cuh"

namespace atlas {

namespace {

constexpr int PR_SMS = 148;
constexpr int PR_THREADS = 16 * 32, PR_MMA = 14, PR_LOAD = 15;   // warps of the roles: softmax, rebuilding, MMA, loads

template <int D>
struct Prompt {
    static constexpr int TILES = D == 256 ? 1 : 2, KEYS = D == 256 ? 64 : 128;
    static constexpr int REBUILD = 4 * TILES, REBUILDERS = 6;   // first warp, warps (half of them keys, half values)
    static constexpr int ROWS = 128 * TILES, SLABS = KEYS / KV_SLAB;
    static constexpr int GROUPS = D / 64, SLAB = kv_slab_bytes(D);
    static constexpr int Q_BYTES = 128 * D * 2;             // a Q tile: D / 64 subtiles of 128 rows of 128 bytes
    static constexpr int KV_BYTES = KEYS * D * 2;           // a K tile: D / 64 subtiles of KEYS rows (tokens); a V tile: KEYS / 64 subtiles of D rows (channels)
    static constexpr int STAGES = 2, RING = D == 64 ? 15 : D == 128 ? 12 : 6;   // rebuilt tiles; halves of slabs, of keys and of values
    static constexpr int HALF = SLAB / 2;                   // codes, then scales and zero points
    static constexpr uint32_t OFF_Q = 0, OFF_K = OFF_Q + TILES * Q_BYTES, OFF_V = OFF_K + STAGES * KV_BYTES, OFF_RAW = OFF_V + STAGES * KV_BYTES;
    static constexpr uint32_t OFF_INFO = OFF_RAW + 2 * RING * HALF, OFF_BAR = OFF_INFO + 16 * 8;
    // barriers; those of S and of O have a place for each of four tiles in a row, so that who comes late can tell them apart
    static constexpr int RAW_FULL = 0, RAW_EMPTY = RAW_FULL + 2 * RING, K_FULL = RAW_EMPTY + 2 * RING, V_FULL = K_FULL + STAGES, S_FULL = V_FULL + STAGES,
                         P_FULL = S_FULL + 8, O_DONE = P_FULL + 2, Q_FULL = O_DONE + 4, DRAIN = Q_FULL + 1, Q_RAW = DRAIN + 1, BARS = Q_RAW + 4 * TILES;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + BARS * 8, TOTAL = OFF_TMEM + 16 + 1024 /* alignment */;
    // columns of tensor memory: O, then S (P over it)
    static constexpr uint32_t T_S = TILES * D, T_COLS = 512;
    static_assert(T_S + 256 <= T_COLS, "tensor memory");
    static_assert(REBUILD + REBUILDERS <= PR_MMA, "warps");
    // A parity tells two rounds of a place apart: who waits for one has to have seen the last, so a place has one lane that fills it and one warp that empties it.
    static_assert(RING <= 16 && RING % (REBUILDERS / 2) == 0, "rounds of the rings");
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};

constexpr uint32_t pr_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void store_transposable(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
// Pairs of fp32 numbers, one instruction for both.
using f32x2 = uint64_t;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// The lowest n bits.
__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
// A wait of a whole (converged) warp: one poll where the phase is over already.
template <int NS = 0>
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const volatile int *abort_flag) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return mbar_wait_warp<NS>(bar, parity, abort_flag);
}

// The tiles of tokens that rows at positions up to p1 see, the first of them at p0.
template <int KEYS>
struct Walk {
    int p1, window_start, sinks, window_tile, sink_tiles, tiles;
    __device__ __forceinline__ Walk(const Attention &a, int p0, int p1) : p1(p1), window_start(0), sinks(0), window_tile(0), sink_tiles(0), tiles(0) {
        if (p1 < 0) return;
        if (a.window) {
            window_start = max(0, p0 - a.window + 1);
            sinks = min(a.sinks, p1 + 1);
            window_tile = window_start / KEYS;
            sink_tiles = min((sinks + KEYS - 1) / KEYS, window_tile);
        }
        tiles = sink_tiles + p1 / KEYS + 1 - window_tile;
    }
    __device__ __forceinline__ int tile(int j) const { return j < sink_tiles ? j : j - sink_tiles + window_tile; }
    // whether a slab has a token that some row sees
    __device__ __forceinline__ bool slab_seen(int s) const { return s * KV_SLAB <= p1 && (s * KV_SLAB + KV_SLAB > window_start || s * KV_SLAB < sinks); }
};

// Query and member of the group of a row, and of rows further on, without another division.
struct RowWalk {
    int query, member;
    __device__ __forceinline__ RowWalk(const Attention &a, int row) : query(row / a.group), member(row - query * a.group) {}
    __device__ __forceinline__ void advance(const Attention &a, int rows) {
        member += rows;
        while (member >= a.group) member -= a.group, ++query;
    }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(PR_THREADS, 1) kv_prompt_kernel(const Attention a, int splits) {
    using P = Prompt<D>;
    constexpr int PR_REBUILD = P::REBUILD, PR_REBUILDERS = P::REBUILDERS;
    constexpr int TILES = P::TILES, KEYS = P::KEYS, SLABS = P::SLABS, STAGES = P::STAGES, RING = P::RING;
    extern __shared__ uint8_t smem_raw[];
    wait_for_front();
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int head = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads / splits, split = blockIdx.x / a.kv_heads % splits;
    // later rows see more: those of all heads and sequences go first
    const int row0 = (int)(gridDim.y - 1 - blockIdx.y) * P::ROWS;
    const Sequence seq = sequence(a, b);
    // (rows that are no sequence's: one warp of each CTA of the sequence next to them)
    auto zero_rest = [&]() {
        zero_rows_next_to(a, seq, b, D, ((int64_t)(split * a.kv_heads + head) * gridDim.y + blockIdx.y) * 32 + lane, (int64_t)splits * a.kv_heads * gridDim.y * 32);
    };
    const int rows = (int)min((int64_t)P::ROWS, (int64_t)seq.served(a) * a.group - row0);
    if (rows <= 0) {
        if (warp == PR_LOAD) zero_rest();
        return;
    }
    const int used = TILES == 2 && rows > 128 ? 2 : 1;   // row tiles with rows
    const int p_first = seq.start() + row0 / a.group, p_last = seq.start() + (row0 + rows - 1) / a.group;
    const Walk<KEYS> walk(a, p_first, p_last);
    const int j0 = (int)((int64_t)walk.tiles * split / splits), tiles = (int)((int64_t)walk.tiles * (split + 1) / splits) - j0;

    const uint32_t raw_base = smem_u32(smem_raw), base = (raw_base + 1023u) & ~1023u;
    uint8_t *const sm = smem_raw + (base - raw_base);
    auto bar = [&](int i) { return base + P::OFF_BAR + 8u * (uint32_t)i; };
    volatile uint32_t *const tmem_slot = reinterpret_cast<volatile uint32_t *>(sm + P::OFF_TMEM);
    volatile int *const s_abort = reinterpret_cast<volatile int *>(sm + P::OFF_TMEM + 8);
    volatile uint8_t *const gone = sm + P::OFF_INFO;   // [tile % 16][slab]: whether the slab is not there

    if (warp == 0) {
        for (int i = lane; i < P::BARS; i += 32)
            mbar_init(bar(i), i >= P::K_FULL && i < P::V_FULL + STAGES ? SLABS : i >= P::P_FULL && i < P::P_FULL + 2 ? 4 : i == P::Q_FULL ? 4 * TILES : 1);
        if (lane < 16) reinterpret_cast<volatile uint64_t *>(gone)[lane] = 0;
        if (lane == 0) *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == PR_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)tmem_slot)), "r"(P::T_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    int issued = 0;              // half slabs that this lane has asked for (loader)
    // S of row tile i (two row tiles), or into buffer j % 2 (one)
    auto s_full = [&](int i, int j) { return bar(P::S_FULL + (TILES == 2 ? 4 * i : 0) + j % 4); };
    auto s_parity = [&](int j) { return (uint32_t)((j / 4) & 1); };

    if (warp == PR_LOAD) {
        // ------------------------------ slabs ------------------------------
        // Lane i brings the slabs' keys that belong in place i of the ring, lane 16 + i the values, as far ahead as there is room.
        const int part = lane / 16, slot = part * RING + lane % 16;
        const bool mine = lane % 16 < RING;
        auto page_of = [&](int n) {
            const int s = walk.tile(j0 + n / SLABS) * SLABS + n % SLABS;
            return n < tiles * SLABS && walk.slab_seen(s) ? a.page_table[b * a.table_stride + s * KV_SLAB / a.page_size] : -1;
        };
        int n = lane % 16, page = mine ? page_of(n) : -1, idle = 0;
        while (true) {
            const bool more = mine && n < tiles * SLABS;
            const bool go = more && (issued == 0 || mbar_try_wait(bar(P::RAW_EMPTY + slot), (uint32_t)((issued - 1) & 1)));
            if (go) {
                const bool there = page >= 0 && page < a.num_pages;
                const int j = n / SLABS, slab = n % SLABS;
                gone[j % 16 * 8 + slab] = !there;
                mbar_arrive_expect_tx(bar(P::RAW_FULL + slot), there ? P::HALF : 0);
                if (there) {
                    const int token = (walk.tile(j0 + j) * SLABS + slab) * KV_SLAB;
                    const uint8_t *src = a.cache + (((int64_t)page * a.kv_heads + head) * (a.page_size / KV_SLAB) + token % a.page_size / KV_SLAB) * P::SLAB;
                    const uint32_t dst = base + P::OFF_RAW + slot * P::HALF;
                    bulk_load_1d(dst, src + part * kv_value_codes(D), 8 * D, bar(P::RAW_FULL + slot));
                    bulk_load_1d(dst + 8 * D, src + (part ? kv_value_params(D) : kv_key_params(D)), D, bar(P::RAW_FULL + slot));
                }
                ++issued;
                n += RING;
                page = page_of(n);
            }
            if (!__any_sync(0xffffffffu, more)) break;
            if (__any_sync(0xffffffffu, go)) {
                idle = 0;
            } else {
                if (++idle > SPIN_LIMIT) *s_abort = 1;
                if (__any_sync(0xffffffffu, *s_abort != 0)) break;
                __nanosleep(100);
            }
        }
        zero_rest();
    } else if (warp >= PR_REBUILD && warp < PR_REBUILD + PR_REBUILDERS) {
        // ------------------------------ codes to fp16: a warp a slab, half of the warps keys, half values ------------------------------
        const int g = lane / 4, t = lane % 4;
        const bool keys = warp < PR_REBUILD + PR_REBUILDERS / 2;
        uint2 w[2][P::GROUPS];   // of both halves of the slab: codes, then scales and zero points
        bool q_done = false;     // the second place of the tiles has Q's rows first
        for (int n = (warp - PR_REBUILD) % (PR_REBUILDERS / 2); n < tiles * SLABS; n += PR_REBUILDERS / 2) {
            const int j = n / SLABS, slab = n % SLABS, slot = (keys ? 0 : RING) + n % RING, st = j % STAGES;
            if (!wait_warp<20>(bar(P::RAW_FULL + slot), (uint32_t)((n / RING) & 1), s_abort)) { *s_abort = 1; break; }
            const uint8_t *src = sm + P::OFF_RAW + slot * P::HALF;
            if (st == 1 && !q_done) {
                if (!wait_warp<20>(bar(P::Q_FULL), 0, s_abort)) { *s_abort = 1; break; }
                q_done = true;
            }
            if (keys) {
                const int spread = (g & 1) * 4 + g / 2;   // eight lanes that store at a time: rows 4 apart, so that the swizzle keeps them apart
                __half2 sb[2][P::GROUPS];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int gr = 0; gr < P::GROUPS; ++gr) {
                        w[h][gr] = *reinterpret_cast<const uint2 *>(src + kv_key_word(D, 8 * h + spread, t + 8 * gr));
                        sb[h][gr] = *reinterpret_cast<const __half2 *>(src + 8 * D + ((8 * h + spread) * P::GROUPS + gr) * 4);
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(P::RAW_EMPTY + slot));
                // the products with the K of this place are done with the last S made of it
                if (j >= STAGES && !wait_warp<20>(s_full(used - 1, j - STAGES), s_parity(j - STAGES), s_abort)) { *s_abort = 1; break; }
                uint8_t *const kt = sm + P::OFF_K + st * P::KV_BYTES;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = slab * KV_SLAB + 8 * h + spread;
#pragma unroll
                    for (int gr = 0; gr < P::GROUPS; ++gr) {
                        const __half2 s = __low2half2(sb[h][gr]), bias = __high2half2(sb[h][gr]), bias16 = minus16_of(bias);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            __half2 v[4];
                            open_word(i ? w[h][gr].y : w[h][gr].x, bias, bias16, v);
                            *reinterpret_cast<uint4 *>(kt + gr * KEYS * 128 + row * 128 + (((4 * i + t) ^ (row & 7)) << 4)) =
                                make_uint4(h2(__hmul2(v[0], s)), h2(__hmul2(v[1], s)), h2(__hmul2(v[2], s)), h2(__hmul2(v[3], s)));
                        }
                    }
                }
            } else {
                uint2 sb[2][P::GROUPS];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int gr = 0; gr < P::GROUPS; ++gr) {
                        w[h][gr] = *reinterpret_cast<const uint2 *>(src + kv_value_unit(D, 8 * h + 2 * t, g + 16 * gr));
                        sb[h][gr] = *reinterpret_cast<const uint2 *>(src + 8 * D + ((4 * h + t) * P::GROUPS + gr) * 8);
                    }
                const bool absent = gone[j % 16 * 8 + slab];
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(P::RAW_EMPTY + slot));
                const int token0 = walk.tile(j0 + j) * KEYS + slab * KV_SLAB;
                if (absent || token0 + KV_SLAB > seq.length || (token0 < walk.window_start && token0 + KV_SLAB > walk.sinks)) {
                    // tokens that no row sees may hold anything: zeros (their weights are zero too, but not times NaN)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int token = token0 + 8 * h + 2 * t;
                        auto seen = [&](int k) { return !absent && k < seq.length && (k >= walk.window_start || k < walk.sinks); };
                        const uint32_t keep = (seen(token) ? 0xffffu : 0u) | (seen(token + 1) ? 0xffff0000u : 0u);
#pragma unroll
                        for (int gr = 0; gr < P::GROUPS; ++gr) sb[h][gr].x &= keep, sb[h][gr].y = (sb[h][gr].y & keep) | (0x64006400u & ~keep);
                    }
                }
                // the product with the V of this place is done with the S after it (with one row tile: it says so itself)
                if (j >= STAGES) {
                    const bool ok = TILES == 2 ? wait_warp<20>(s_full(used - 1, j - STAGES + 1), s_parity(j - STAGES + 1), s_abort)
                                               : wait_warp<20>(bar(P::O_DONE + (j - STAGES) % 4), s_parity(j - STAGES), s_abort);
                    if (!ok) { *s_abort = 1; break; }
                }
                const uint32_t vt = base + P::OFF_V + st * P::KV_BYTES + (slab / 4) * (D * 128);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int gr = 0; gr < P::GROUPS; ++gr) {
                        const __half2 s = h2(sb[h][gr].x), bias = h2(sb[h][gr].y), bias16 = minus16_of(bias);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            __half2 v[4];
                            open_word(i ? w[h][gr].y : w[h][gr].x, bias, bias16, v);
                            // row 32 j + 8 p + g of the tile is channel 32 j + 4 g + p: eight neighbouring rows a matrix
                            store_transposable(vt + (uint32_t)((32 * (2 * gr + i) + lane) * 128 + (((2 * (slab % 4) + h) ^ (lane & 7)) << 4)), h2(__hmul2(v[0], s)),
                                               h2(__hmul2(v[1], s)), h2(__hmul2(v[2], s)), h2(__hmul2(v[3], s)));
                        }
                    }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar((keys ? P::K_FULL : P::V_FULL) + st));
        }
    } else if (warp == PR_MMA) {
        // ------------------------------ MMAs ------------------------------
        const uint64_t dq0 = make_smem_desc(base + P::OFF_Q), dk0 = make_smem_desc(base + P::OFF_K), dv0 = make_smem_desc(base + P::OFF_V);
        bool ok = tiles == 0 || wait_warp(bar(P::Q_FULL), 0, s_abort);
        auto qk = [&](int j, int tile, int buffer) {   // the address field counts 16-byte units
            const uint64_t dk = dk0 + (uint64_t)((j % STAGES) * (P::KV_BYTES >> 4)), dq = dq0 + (uint64_t)(tile * (P::Q_BYTES >> 4));
            const uint32_t d = tmem + P::T_S + buffer * KEYS, done = s_full(tile, j);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    umma_f16_ss(d, dq + (uint64_t)((k / 4) * 1024 + (k % 4) * 2), dk + (uint64_t)((k / 4) * (KEYS * 8) + (k % 4) * 2), pr_idesc(KEYS), k != 0);
                umma_commit(done);
            }
        };
        auto pv = [&](int j, int tile, int buffer) {
            const uint64_t dv = dv0 + (uint64_t)((j % STAGES) * (P::KV_BYTES >> 4));
            const uint32_t d = tmem + tile * D, p = tmem + P::T_S + buffer * KEYS;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < KEYS / 16; ++k)
                    umma_f16_ts(d, p + k * 8, dv + (uint64_t)((k / 4) * (D * 8) + (k % 4) * 2), pr_idesc(D), k != 0 ? 1u : (uint32_t)(j != 0));
            }
        };
        auto commit = [&](uint32_t at) { if (elect_one()) umma_commit(at); };
        if constexpr (TILES == 2) {
            // S of a row tile is written behind the product that has read P from the same columns: the tensor core works in order
            for (int j = 0; j <= tiles && ok && tiles; ++j) {
                if (j < tiles) ok = wait_warp(bar(P::K_FULL + j % STAGES), (uint32_t)((j / STAGES) & 1), s_abort);
                if (ok && j > 0) ok = wait_warp(bar(P::V_FULL + (j - 1) % STAGES), (uint32_t)(((j - 1) / STAGES) & 1), s_abort);
                for (int i = 0; i < used && ok; ++i) {
                    if (j > 0) ok = wait_warp(bar(P::P_FULL + i), (uint32_t)((j - 1) & 1), s_abort);
                    if (!ok) break;
                    tcgen05_fence_after();
                    if (j > 0) pv(j - 1, i, i);
                    if (j < tiles) qk(j, i, i);
                }
            }
            if (ok && tiles) commit(bar(P::O_DONE));
        } else {
            for (int j = -1; j < tiles && ok && tiles; ++j) {
                if (j + 1 < tiles) {
                    ok = wait_warp(bar(P::K_FULL + (j + 1) % STAGES), (uint32_t)(((j + 1) / STAGES) & 1), s_abort);
                    if (!ok) break;
                    tcgen05_fence_after();
                    qk(j + 1, 0, (j + 1) & 1);
                }
                if (j >= 0) {
                    ok = wait_warp(bar(P::V_FULL + j % STAGES), (uint32_t)((j / STAGES) & 1), s_abort) &&
                         wait_warp(bar(P::P_FULL + (j & 1)), (uint32_t)((j / 2) & 1), s_abort);
                    if (!ok) break;
                    tcgen05_fence_after();
                    pv(j, 0, j & 1);
                    commit(bar(P::O_DONE + j % 4));
                }
            }
        }
        if (!ok) *s_abort = 1;
    } else if (warp < PR_REBUILD) {
        const int tile = warp / 4, in_block = tid, quarter = warp % 4;
        const int row = row0 + in_block, query = row / a.group;
        const bool live = in_block < rows;
        bool ok = true;
        // ------------------------------ Q: a thread a row ------------------------------
        // (Rows come by bulk copies, into the second place of the rebuilt tiles, and go to their own swizzled and as fp16.  Loads by
        // the threads took 10000 cycles of a CTA's first 17000.)
        float factor = fabsf(a.scale_log2);
        {
            static_assert(P::ROWS == 2 * KEYS, "the rows of Q in the places of a K and a V tile");
            constexpr int PIECES = D / 8;
            uint8_t *const raw = sm + (in_block < KEYS ? P::OFF_K : P::OFF_V) + P::KV_BYTES + (in_block % KEYS) * (D * 2);
            uint8_t *const qr = sm + P::OFF_Q + tile * P::Q_BYTES + (in_block % 128) * 128;
            const uint32_t at = bar(P::Q_RAW + warp);
            if (lane == 0) mbar_arrive_expect_tx(at, (uint32_t)min(max(rows - warp * 32, 0), 32) * (D * 2));
            __syncwarp();
            // (rows that lie behind one another, the heads of a token, in one copy: one takes some 36 cycles however small)
            const int member = row - query * a.group, run = a.q_head_stride == D * 2 ? a.group : 1;
            if (live && (run == 1 || member == 0 || lane == 0))
                bulk_load_1d(smem_u32(raw), a.q + (int64_t)(seq.first_query + query) * a.q_token_stride + (head * a.group + member) * a.q_head_stride,
                             min(min(run == 1 ? 1 : run - member, 32 - lane), rows - in_block) * (D * 2), at);
            ok = wait_warp<20>(at, 0, s_abort);
            const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;   // a negative scale turns the queries round: maxima of scores are maxima of products
            float down = 1.0f;
            if (BF16) {
                // times a power of two, so that the largest is in [1, 2): exact, but for numbers below 2^-14 of it, which
                // are off by 2^-25 of it at most
                float top = 0.0f;
                if (live)
#pragma unroll 4
                    for (int c = 0; c < PIECES; ++c) {   // (from another piece in every lane: their banks differ)
                        const uint4 v = *reinterpret_cast<const uint4 *>(raw + (c + lane) % PIECES * 16);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u))));
                    }
                const int ex = min(max((__float_as_int(top) >> 23) & 0xff, 8), 246);
                down = __int_as_float((254 - ex) << 23);
                factor *= __int_as_float(ex << 23);
            }
#pragma unroll 4
            for (int i = 0; i < PIECES; ++i) {
                const int c = (i + lane) % PIECES;
                const uint4 v = live ? *reinterpret_cast<const uint4 *>(raw + c * 16) : make_uint4(0, 0, 0, 0);
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = flip ^ (BF16 ? h2(__floats2half2_rn(__uint_as_float(w[k] << 16) * down, __uint_as_float(w[k] & 0xffff0000u) * down)) : w[k]);
                *reinterpret_cast<uint4 *>(qr + (c / 8) * (128 * 128) + (((c % 8) ^ (in_block & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P::Q_FULL));
        }
        factor = fmaxf(factor, 1e-30f);   // (of a scale of zero: masked scores stay -inf)

        // ------------------------------ softmax: a thread a row ------------------------------
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const int place = live ? seq.start() + query : -1;
        // first and last position of this row tile, for tiles that need no mask
        const int t_first = seq.start() + (row0 + tile * 128) / a.group;
        const int t_last = min(p_last, seq.start() + (row0 + tile * 128 + 127) / a.group);
        const uint32_t t_out = tmem + lanes + tile * D;
        const f32x2 factor2 = pair(factor, factor);
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < tiles && tile < used && ok; ++j) {
            const int buffer = TILES == 2 ? tile : j & 1;
            if (!wait_warp(s_full(tile, j), s_parity(j), s_abort)) { ok = false; break; }
            tcgen05_fence_after();
            const uint32_t ts = tmem + lanes + P::T_S + buffer * KEYS;
            const int token0 = walk.tile(j0 + j) * KEYS;
            const uint64_t absent = reinterpret_cast<volatile uint64_t *>(gone)[j % 16];   // a byte a slab
            if (absent || token0 + KEYS - 1 > t_first || (a.window && token0 <= t_last - a.window && token0 + KEYS > a.sinks)) {
                // -inf where tokens are hidden
#pragma unroll 1
                for (int c = 0; c < SLABS; ++c) {
                    uint32_t v[16];
                    tmem_ld_32x32b_x16(ts + 16 * c, v);
                    const int t0 = token0 + 16 * c;
                    uint32_t seen = first_bits(place + 1 - t0);
                    if (a.window) seen &= ~first_bits(place - a.window + 1 - t0) | first_bits(a.sinks - t0);
                    if ((absent >> (8 * c)) & 0xff) seen = 0;
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = (seen >> i) & 1 ? v[i] : 0xff800000u;
                    tmem_st_32x32b_x16(ts + 16 * c, v);
                }
                tmem_st_wait();
            }
            // the maximum
            float tops[2] = {-INFINITY, -INFINITY};
            uint32_t s[2][32];
            tmem_ld_32x32b_x32(ts, s[0]);
#pragma unroll 1
            for (int c = 0; c < KEYS; c += 64) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    tmem_ld_wait();
                    if (e == 0 || c + 64 < KEYS) tmem_ld_32x32b_x32(ts + c + 32 * (e + 1), s[e ^ 1]);
#pragma unroll
                    for (int i = 0; i < 16; ++i) tops[i & 1] = fmaxf(tops[i & 1], fmaxf(__uint_as_float(s[e][2 * i]), __uint_as_float(s[e][2 * i + 1])));
                }
            }
            const float top = fmaxf(tops[0], tops[1]) * factor;
            if (__any_sync(0xffffffffu, top > m + KV_HEADROOM)) {   // rare, but for the first tile: what there is shrinks
                const float now = fmaxf(m, top), shrink = m == -INFINITY ? 0.0f : exp2_fast(m - now);
                m = now;
                l *= shrink;
                if (j > 0) {
                    // (two row tiles: S of this tile came behind the product into O)
                    if (TILES == 1 && !wait_warp(bar(P::O_DONE + (j - 1) % 4), s_parity(j - 1), s_abort)) { ok = false; break; }
                    tcgen05_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(t_out + c * 16, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                        tmem_st_32x32b_x16(t_out + c * 16, o);
                    }
                }
            }
            // the weights, over what has been read of S
            const float ref = m == -INFINITY ? 0.0f : KV_SHIFT - m;
            const f32x2 ref2 = pair(ref, ref);
            f32x2 sums = pair(0.0f, 0.0f);
            tmem_ld_32x32b_x32(ts, s[0]);
#pragma unroll 1
            for (int c = 0; c < KEYS; c += 64) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    tmem_ld_wait();
                    if (e == 0 || c + 64 < KEYS) tmem_ld_32x32b_x32(ts + c + 32 * (e + 1), s[e ^ 1]);
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x, y;
                        unpair(fma2(pair(__uint_as_float(s[e][2 * i]), __uint_as_float(s[e][2 * i + 1])), factor2, ref2), x, y);
                        x = exp2_fast(x), y = exp2_fast(y);
                        sums = add2(sums, pair(x, y));
                        p[i] = h2(__floats2half2_rn(x, y));
                    }
                    tmem_st_32x32b_x16(ts + c / 2 + 16 * e, p);
                }
            }
            float even, odd;
            unpair(sums, even, odd);
            l += even + odd;
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P::P_FULL + buffer));
        }
        // ------------------------------ output ------------------------------
        if (ok && tiles && tile < used) ok = wait_warp(bar(P::O_DONE + (TILES == 2 ? 0 : (tiles - 1) % 4)), TILES == 2 ? 0u : s_parity(tiles - 1), s_abort);
        if (!ok) *s_abort = 1;
        if (__all_sync(0xffffffffu, ok) && tile < used) {
            tcgen05_fence_after();
            const float inv = splits > 1 ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
            // (a split leaves maximum, sum and output of each row)
            float *part = a.partial + ((((int64_t)b * splits + split) * a.kv_heads + head) * gridDim.y * P::ROWS + row) * (D + 4);
            if (splits > 1 && live) *reinterpret_cast<float2 *>(part) = make_float2(m, l);
            // rows go out whole, by way of Q's place, which nothing reads any more: this warp's rows, their 16-byte pieces shifted by row
            constexpr int PIECES = D / 8;
            uint8_t *const stage = sm + P::OFF_Q + warp * (32 * D * 2);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (tiles) {
                    tmem_ld_32x32b_x32(t_out + c * 32, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                auto at = [&](int ch) { return __uint_as_float(o[8 * (ch % 4) + ch / 4]) * inv; };   // channel 32 c + ch
                if (splits > 1) {
                    if (live)
#pragma unroll
                        for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(part + 4 + c * 32 + 4 * i) = make_float4(at(4 * i), at(4 * i + 1), at(4 * i + 2), at(4 * i + 3));
                } else if (tiles) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 x = pack4<BF16>(at(8 * i), at(8 * i + 1), at(8 * i + 2), at(8 * i + 3)), y = pack4<BF16>(at(8 * i + 4), at(8 * i + 5), at(8 * i + 6), at(8 * i + 7));
                        *reinterpret_cast<uint4 *>(stage + lane * (D * 2) + (((c * 4 + i) ^ (lane % 8)) << 4)) = make_uint4(x.x, x.y, y.x, y.y);
                    }
                }
            }
            if (splits == 1) {
                __syncwarp();
                const int piece = lane % PIECES;
                RowWalk at(a, row0 + warp * 32 + lane / PIECES);
#pragma unroll 2
                for (int r = lane / PIECES; r < 32; r += 32 / PIECES) {
                    if (warp * 32 + r < rows)
                        *reinterpret_cast<uint4 *>(a.out + (((int64_t)(seq.first_query + at.query) * a.q_heads + head * a.group + at.member) * (int64_t)D + piece * 8) * 2) =
                            tiles ? *reinterpret_cast<const uint4 *>(stage + r * (D * 2) + ((piece ^ (r % 8)) << 4)) : make_uint4(0, 0, 0, 0);
                    at.advance(a, 32 / PIECES);
                }
            }
        }
        tcgen05_fence_before();
    }

    __syncthreads();
    if (*s_abort) {
        // a wait ran out somewhere: no copy may land, and no MMA run, once this CTA has gone
        if (warp == PR_LOAD && issued > 0) mbar_wait<100>(bar(P::RAW_FULL + lane / 16 * RING + lane % 16), (uint32_t)((issued - 1) & 1));
        if (warp < PR_REBUILD) mbar_wait<100>(bar(P::Q_RAW + warp), 0);
        if (warp == PR_MMA && lane == 0) {
            umma_commit(bar(P::DRAIN));
            mbar_wait<100>(bar(P::DRAIN), 0);
            if (a.status) *a.status = 1;
        }
        __syncthreads();
    }
    tcgen05_fence_after();
    if (warp == PR_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::T_COLS) : "memory");
}

// Joins the splits of a row, in order.  A thread makes four channels.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) kv_prompt_join_kernel(const Attention a, int splits, int blocks) {
    using P = Prompt<D>;
    const int b = blockIdx.z, head = blockIdx.y, x = blockIdx.x * 256 + threadIdx.x, row = x / (D / 4), c = x % (D / 4) * 4;
    const Sequence seq = sequence(a, b);
    char *dst = out_row(a, seq, head, row, D);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!dst) return;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < splits; ++s) {
        const float *part = a.partial + ((((int64_t)b * splits + s) * a.kv_heads + head) * blocks * P::ROWS + row) * (D + 4);
        const float2 ml = *reinterpret_cast<const float2 *>(part);
        const float4 po = *reinterpret_cast<const float4 *>(part + 4 + c);
        const float top = fmaxf(m, ml.x);
        const float wa = m == -INFINITY ? 0.0f : exp2_fast(m - top), wb = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top);
        l = l * wa + ml.y * wb;
        o.x = o.x * wa + po.x * wb, o.y = o.y * wa + po.y * wb, o.z = o.z * wa + po.z * wb, o.w = o.w * wa + po.w * wb;
        m = top;
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    *reinterpret_cast<uint2 *>(dst + c * 2) = pack4<BF16>(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

struct PromptPlan {
    int64_t blocks;              // row blocks of a sequence and head
    int splits;
    size_t bytes;
};
PromptPlan plan_of(const AtlasKvAttention &p) {
    PromptPlan plan;
    const int64_t rows = p.max_queries * (p.q_heads / p.kv_heads), block = p.head_dim == 256 ? 128 : 256;
    plan.blocks = ceil_div_i64(std::max<int64_t>(rows, 1), block);
    // CTAs for most SMs: the tokens are split where there are few row blocks, into parts of four tiles at least.
    const int64_t ctas = plan.blocks * p.kv_heads * p.batch, tiles = p.max_pages * p.page_size / 128;
    plan.splits = (int)std::max<int64_t>(1, std::min<int64_t>({PR_SMS / std::max<int64_t>(ctas, 1), tiles / 4, 16}));
    plan.bytes = plan.splits > 1 ? (size_t)(p.batch * plan.splits * p.kv_heads * plan.blocks * block * (p.head_dim + 4) * 4) : 0;
    return plan;
}

template <int D, bool BF16>
int launch(const Attention &a, const PromptPlan &plan, cudaStream_t stream) {
    using P = Prompt<D>;
    const char *what = "atlas_kv_attention";
    auto *kernel = kv_prompt_kernel<D, BF16>;
    int e = allow_smem<kv_prompt_kernel<D, BF16>>(P::TOTAL, what);
    if (e == ATLAS_OK) e = launch_early(kernel, dim3((unsigned)(a.batch * plan.splits * a.kv_heads), (unsigned)plan.blocks), PR_THREADS, P::TOTAL, stream, what, a, plan.splits);
    if (e != ATLAS_OK || plan.splits == 1) return e;
    return launch_early(kv_prompt_join_kernel<D, BF16>, dim3((unsigned)(plan.blocks * P::ROWS * (D / 4) / 256), (unsigned)a.kv_heads, (unsigned)a.batch), 256, 0, stream, what, a,
                        plan.splits, (int)plan.blocks);
}

}  // namespace

// From 33 rows of a kv head on (25 of 256 channels): 8 sequences of 4000 tokens on 8 kv heads, 48 rows of 128 channels 45 us and
// 55 by kv_attention_kernel, 32 rows 44 and 41; 32 rows of 256 channels (4 of 8000 on 2) 32 and 48, 16 rows 29 and 34.
bool kv_prompt_serves(const AtlasKvAttention &p) {
    return p.max_queries * (p.q_heads / p.kv_heads) > (p.head_dim == 256 ? 24 : 32) && p.batch * p.kv_heads <= (1 << 20);
}

int64_t kv_prompt_blocks(const AtlasKvAttention &p) { return plan_of(p).blocks; }

size_t kv_prompt_workspace_bytes(const AtlasKvAttention &p) { return plan_of(p).bytes; }

int kv_prompt(const Attention &a, const AtlasKvAttention &p, cudaStream_t stream) {
    const PromptPlan plan = plan_of(p);
    const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
    switch (p.head_dim) {
        case 64: return bf16 ? launch<64, true>(a, plan, stream) : launch<64, false>(a, plan, stream);
        case 128: return bf16 ? launch<128, true>(a, plan, stream) : launch<128, false>(a, plan, stream);
        default: return bf16 ? launch<256, true>(a, plan, stream) : launch<256, false>(a, plan, stream);
    }
}

}  // namespace atlas
