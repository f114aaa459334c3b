// Attention of many queries over the 4-bit cache (prompts, chunks of prompts) on the tensor cores.
//
// A CTA takes one kv head and TILES tiles of 128 rows (queries x the query heads that share the kv head) and walks the
// tiles of 64 tokens that any of them sees:
//   S = Q K^T      tcgen05, M 128 rows, N 64 tokens; Q stays in tensor memory as fp16 (bf16 rows times a power of two)
//   P = 2^(S' - m) a thread a row; P goes back to tensor memory as fp16, over S
//   O += P V       tcgen05, A from tensor memory, N = D channels, fp32 accumulators in tensor memory
// K and V are rebuilt from their codes into 128-byte-swizzled K-major tiles in shared memory, as the exact fp16 numbers that
// the cache stands for, so the only roundings are those of P and of the output.  The running maximum of a row follows its
// scores only where they pass it by 2^8 (O is rescaled then, which is rare); P keeps 14 bits of headroom for that.
//
// Warps: 0-3 and 4-7 softmax of the two row tiles (of one tile if D is 256, where O takes the tensor memory of both; its S
// then has two buffers), 8-11 rebuild, 12 issues the MMAs, 13 brings slabs in by bulk copies.  While the softmax warps of one
// row tile work, the tensor core works on the other.
#include <algorithm>

#include "kv_attention.cuh"

namespace atlas {

namespace {

constexpr int PR_KEYS = 64, PR_THREADS = 14 * 32;
constexpr int PR_REBUILD = 8, PR_MMA = 12, PR_LOAD = 13;   // first warps of the roles

template <int D>
struct Prompt {
    static constexpr int TILES = D == 256 ? 1 : 2;
    static constexpr int ROWS = 128 * TILES;
    static constexpr int GROUPS = D / 64, SLAB = kv_slab_bytes(D);
    static constexpr int KV_BYTES = PR_KEYS * D * 2;        // a K tile: D / 64 subtiles of 64 rows (tokens); a V tile: D rows (channels)
    static constexpr int KS = D == 256 ? 2 : 3, RS = D == 256 ? 2 : 4;   // stages: rebuilt tiles, raw tiles
    static constexpr int RAW_BYTES = 4 * SLAB;
    static constexpr uint32_t OFF_K = 0, OFF_V = OFF_K + KS * KV_BYTES, OFF_RAW = OFF_V + KS * KV_BYTES, OFF_INFO = OFF_RAW + RS * RAW_BYTES;
    static constexpr uint32_t OFF_BAR = OFF_INFO + 16 * 4;
    // barriers
    static constexpr int RAW_FULL = 0, RAW_EMPTY = RAW_FULL + RS, K_FULL = RAW_EMPTY + RS, K_EMPTY = K_FULL + KS, V_FULL = K_EMPTY + KS, V_EMPTY = V_FULL + KS,
                         S_FULL = V_EMPTY + KS, P_FULL = S_FULL + 2, O_DONE = P_FULL + 2, Q_FULL = O_DONE + 1, DRAIN = Q_FULL + 1,
                         BARS = DRAIN + 1;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + BARS * 8, TOTAL = OFF_TMEM + 16 + 1024 /* alignment */;
    // columns of tensor memory: O, then S (P over it), then Q
    static constexpr uint32_t T_S = TILES * D, T_Q = T_S + 2 * PR_KEYS, T_COLS = 512;
    static_assert(T_Q + TILES * D / 2 <= T_COLS, "tensor memory");
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

// The tiles of 64 tokens that rows p0 .. p1 (positions) see.
struct Walk {
    int p1, window_start, sinks, window_tile, sink_tiles, tiles;
    __device__ __forceinline__ int tile(int j) const { return j < sink_tiles ? j : j - sink_tiles + window_tile; }
    // whether a slab has a token that some row sees
    __device__ __forceinline__ bool slab_seen(int s) const { return s * KV_SLAB <= p1 && (s * KV_SLAB + KV_SLAB > window_start || s * KV_SLAB < sinks); }
};
__device__ __forceinline__ Walk make_walk(const Attention &a, int p0, int p1) {
    Walk w = {p1, 0, 0, 0, 0, 0};
    if (p1 < 0) return w;
    if (a.window) {
        w.window_start = max(0, p0 - a.window + 1);
        w.sinks = min(a.sinks, p1 + 1);
        w.window_tile = w.window_start / PR_KEYS;
        w.sink_tiles = min((w.sinks + PR_KEYS - 1) / PR_KEYS, w.window_tile);
    }
    w.tiles = w.sink_tiles + p1 / PR_KEYS + 1 - w.window_tile;
    return w;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(PR_THREADS, 1) kv_prompt_kernel(const Attention a, int splits) {
    using P = Prompt<D>;
    constexpr int KS = P::KS, RS = P::RS, TILES = P::TILES;
    extern __shared__ uint8_t smem_raw[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int b = blockIdx.z / splits, split = blockIdx.z % splits, head = blockIdx.y;
    // later rows see more: they go first
    const int row0 = (int)(gridDim.x - 1 - blockIdx.x) * P::ROWS;
    const Sequence seq = sequence(a, b);
    const int rows = (int)min((int64_t)P::ROWS, (int64_t)seq.queries * a.group - row0);
    if (rows <= 0) return;
    const int p_first = seq.length - seq.queries + row0 / a.group, p_last = seq.length - seq.queries + (row0 + rows - 1) / a.group;
    const Walk walk = make_walk(a, p_first, p_last);
    const int j0 = (int)((int64_t)walk.tiles * split / splits), tiles = (int)((int64_t)walk.tiles * (split + 1) / splits) - j0;

    const uint32_t raw_base = smem_u32(smem_raw), base = (raw_base + 1023u) & ~1023u;
    uint8_t *const sm = smem_raw + (base - raw_base);
    auto bar = [&](int i) { return base + P::OFF_BAR + 8u * (uint32_t)i; };
    volatile uint32_t *const tmem_slot = reinterpret_cast<volatile uint32_t *>(sm + P::OFF_TMEM);
    volatile int *const s_abort = reinterpret_cast<volatile int *>(sm + P::OFF_TMEM + 8);
    volatile uint32_t *const info = reinterpret_cast<volatile uint32_t *>(sm + P::OFF_INFO);   // slabs of a tile that are not there

    if (tid == 0) {
        for (int i = 0; i < RS; ++i) mbar_init(bar(P::RAW_FULL + i), 1), mbar_init(bar(P::RAW_EMPTY + i), 4);
        for (int i = 0; i < KS; ++i) {
            mbar_init(bar(P::K_FULL + i), 4), mbar_init(bar(P::K_EMPTY + i), 1);
            mbar_init(bar(P::V_FULL + i), 4), mbar_init(bar(P::V_EMPTY + i), 1);
        }
        for (int i = 0; i < 2; ++i) mbar_init(bar(P::S_FULL + i), 1), mbar_init(bar(P::P_FULL + i), 4);
        mbar_init(bar(P::O_DONE), 1);
        mbar_init(bar(P::Q_FULL), 4 * TILES);
        mbar_init(bar(P::DRAIN), 1);
        *s_abort = 0;
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
    int issued = 0;              // raw tiles asked for (loader), MMA groups committed (MMA warp)

    if (warp == PR_LOAD) {
        // ------------------------------ slabs ------------------------------
        int pages = -1;          // lane i: page of slab i % 4 of tile i / 4 of this batch of 8 tiles
        bool pages_seen = false;
        for (int j = 0; j < tiles; ++j) {
            if (j % 8 == 0) {
                const int jj = j + lane / 4, s = walk.tile(j0 + jj) * 4 + lane % 4;
                pages_seen = jj < tiles && walk.slab_seen(s);
                pages = pages_seen ? a.page_table[b * a.table_stride + s * KV_SLAB / a.page_size] : -1;
            }
            const int stage = j % RS;
            if (j >= RS && !mbar_wait_warp<20>(bar(P::RAW_EMPTY + stage), (uint32_t)((j / RS - 1) & 1), s_abort)) { *s_abort = 1; break; }
            const int from = (j % 8) * 4 + lane % 4, page = __shfl_sync(0xffffffffu, pages, from);
            const bool there = page >= 0 && page < a.num_pages;
            const uint32_t present = __ballot_sync(0xffffffffu, there && lane < 4);
            if (lane == 0) {
                info[j % 16] = ~present & 15u;
                mbar_arrive_expect_tx(bar(P::RAW_FULL + stage), (uint32_t)__popc(present) * P::SLAB);
            }
            __syncwarp();
            if (lane < 4 && there) {
                const int token = (walk.tile(j0 + j) * 4 + lane) * KV_SLAB;
                const uint8_t *src = a.cache + (((int64_t)page * a.kv_heads + head) * (a.page_size / KV_SLAB) + token % a.page_size / KV_SLAB) * P::SLAB;
                bulk_load_1d(base + P::OFF_RAW + stage * P::RAW_BYTES + lane * P::SLAB, src, P::SLAB, bar(P::RAW_FULL + stage));
            }
            issued = j + 1;
        }
    } else if (warp >= PR_REBUILD && warp < PR_MMA) {
        // ------------------------------ codes to fp16 ------------------------------
        const int slab = warp - PR_REBUILD, g = lane / 4, t = lane % 4;
        const int spread = (g & 1) * 4 + g / 2;   // eight lanes that store at a time: rows 4 apart, so that the swizzle keeps them apart
        for (int j = 0; j < tiles; ++j) {
            const int rs = j % RS, ks = j % KS;
            if (!mbar_wait_warp<20>(bar(P::RAW_FULL + rs), (uint32_t)((j / RS) & 1), s_abort)) { *s_abort = 1; break; }
            const uint8_t *src = sm + P::OFF_RAW + rs * P::RAW_BYTES + slab * P::SLAB;
            const bool absent = (info[j % 16] >> slab) & 1;
            const int token0 = walk.tile(j0 + j) * PR_KEYS + slab * KV_SLAB;
            if (j >= KS && !mbar_wait_warp<20>(bar(P::K_EMPTY + ks), (uint32_t)((j / KS - 1) & 1), s_abort)) { *s_abort = 1; break; }
            uint8_t *const kt = sm + P::OFF_K + ks * P::KV_BYTES;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int token = 8 * h + spread, row = slab * KV_SLAB + token;
#pragma unroll
                for (int gr = 0; gr < P::GROUPS; ++gr) {
                    const __half2 sb = *reinterpret_cast<const __half2 *>(src + kv_key_params(D) + (token * P::GROUPS + gr) * 4);
                    const __half2 s = __low2half2(sb), bias = __high2half2(sb), bias16 = __hsub2(bias, __float2half2_rn(960.0f));
                    const uint2 w = *reinterpret_cast<const uint2 *>(src + kv_key_word(D, token, t + 8 * gr));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        __half2 v[4];
                        open_word(i ? w.y : w.x, bias, bias16, v);
                        *reinterpret_cast<uint4 *>(kt + gr * 8192 + row * 128 + (((4 * i + t) ^ (row & 7)) << 4)) =
                            make_uint4(h2(__hmul2(v[0], s)), h2(__hmul2(v[1], s)), h2(__hmul2(v[2], s)), h2(__hmul2(v[3], s)));
                    }
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P::K_FULL + ks));
            if (j >= KS && !mbar_wait_warp<20>(bar(P::V_EMPTY + ks), (uint32_t)((j / KS - 1) & 1), s_abort)) { *s_abort = 1; break; }
            const uint32_t vt = base + P::OFF_V + ks * P::KV_BYTES;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // tokens that are not there may hold anything: zeros (their weights are zero too, but not times NaN)
                uint32_t keep = 0xffffffffu;
                const int token = token0 + 8 * h + 2 * t;
                if (absent || token0 + KV_SLAB > seq.length)
                    keep = absent ? 0u : (token < seq.length ? 0xffffu : 0u) | (token + 1 < seq.length ? 0xffff0000u : 0u);
#pragma unroll
                for (int gr = 0; gr < P::GROUPS; ++gr) {
                    uint2 sb = *reinterpret_cast<const uint2 *>(src + kv_value_params(D) + ((4 * h + t) * P::GROUPS + gr) * 8);
                    sb.x &= keep;
                    sb.y = (sb.y & keep) | (0x64006400u & ~keep);
                    const __half2 s = h2(sb.x), bias = h2(sb.y), bias16 = __hsub2(bias, __float2half2_rn(960.0f));
                    const uint2 w = *reinterpret_cast<const uint2 *>(src + kv_value_codes(D) + kv_value_unit(D, 8 * h + 2 * t, g + 16 * gr));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        __half2 v[4];
                        open_word(i ? w.y : w.x, bias, bias16, v);
                        // row 32 j + 8 p + g of the tile is channel 32 j + 4 g + p: eight neighbouring rows a matrix
                        store_transposable(vt + (uint32_t)((32 * (2 * gr + i) + lane) * 128 + (((2 * slab + h) ^ (lane & 7)) << 4)), h2(__hmul2(v[0], s)), h2(__hmul2(v[1], s)),
                                           h2(__hmul2(v[2], s)), h2(__hmul2(v[3], s)));
                    }
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(P::V_FULL + ks));
                mbar_arrive(bar(P::RAW_EMPTY + rs));
            }
        }
    } else if (warp == PR_MMA) {
        // ------------------------------ MMAs ------------------------------
        const uint64_t dk0 = make_smem_desc(base + P::OFF_K), dv0 = make_smem_desc(base + P::OFF_V);
        bool ok = tiles == 0 || mbar_wait_warp(bar(P::Q_FULL), 0, s_abort);
        auto qk = [&](int j, int tile, int buffer) {   // the address field counts 16-byte units
            const uint64_t dk = dk0 + (uint64_t)((j % KS) * (P::KV_BYTES >> 4));
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    umma_f16_ts(tmem + P::T_S + buffer * PR_KEYS, tmem + P::T_Q + tile * (D / 2) + k * 8, dk + (uint64_t)((k / 4) * 512 + (k % 4) * 2), pr_idesc(PR_KEYS), k != 0);
                umma_commit(bar(P::S_FULL + buffer));
            }
        };
        auto pv = [&](int j, int tile, int buffer) {
            const uint64_t dv = dv0 + (uint64_t)((j % KS) * (P::KV_BYTES >> 4));
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < PR_KEYS / 16; ++k)
                    umma_f16_ts(tmem + tile * D, tmem + P::T_S + buffer * PR_KEYS + k * 8, dv + (uint64_t)(k * 2), pr_idesc(D), (j | k) != 0);
            }
        };
        auto commit = [&](int i) { if (elect_one()) umma_commit(bar(i)); };
        if constexpr (TILES == 2) {
            // S of a row tile is written behind the product that has read P from the same columns: the tensor core works in order
            for (int j = 0; j <= tiles && ok && tiles; ++j) {
                if (j < tiles) ok = mbar_wait_warp(bar(P::K_FULL + j % KS), (uint32_t)((j / KS) & 1), s_abort);
                if (ok && j > 0) ok = mbar_wait_warp(bar(P::V_FULL + (j - 1) % KS), (uint32_t)(((j - 1) / KS) & 1), s_abort);
                for (int i = 0; i < 2 && ok; ++i) {
                    if (j > 0) {
                        ok = mbar_wait_warp(bar(P::P_FULL + i), (uint32_t)((j - 1) & 1), s_abort);
                        if (!ok) break;
                        tcgen05_fence_after();
                        pv(j - 1, i, i);
                    } else {
                        tcgen05_fence_after();
                    }
                    if (j < tiles) qk(j, i, i);
                }
                if (ok && j > 0) commit(P::V_EMPTY + (j - 1) % KS);
                if (ok && j < tiles) commit(P::K_EMPTY + j % KS);
                __syncwarp();
            }
            if (ok && tiles) commit(P::O_DONE);
        } else {
            for (int j = -1; j < tiles && ok && tiles; ++j) {
                if (j + 1 < tiles) {
                    ok = mbar_wait_warp(bar(P::K_FULL + (j + 1) % KS), (uint32_t)(((j + 1) / KS) & 1), s_abort);
                    if (!ok) break;
                    tcgen05_fence_after();
                    qk(j + 1, 0, (j + 1) & 1);
                    commit(P::K_EMPTY + (j + 1) % KS);
                }
                if (j >= 0) {
                    ok = mbar_wait_warp(bar(P::V_FULL + j % KS), (uint32_t)((j / KS) & 1), s_abort) &&
                         mbar_wait_warp(bar(P::P_FULL + (j & 1)), (uint32_t)((j / 2) & 1), s_abort);
                    if (!ok) break;
                    tcgen05_fence_after();
                    pv(j, 0, j & 1);
                    commit(P::V_EMPTY + j % KS);
                    commit(P::O_DONE);
                }
                __syncwarp();
            }
        }
        if (!ok) *s_abort = 1;
    } else if (warp < 4 * TILES) {
        // ------------------------------ softmax: a thread a row ------------------------------
        const int tile = warp / 4, in_block = tid, row = row0 + in_block, query = row / a.group;
        const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
        const bool live = in_block < rows;
        const int place = live ? seq.length - seq.queries + query : -1;
        // first and last position of this row tile, for tiles that need no mask
        const int t_first = seq.length - seq.queries + (row0 + tile * 128) / a.group;
        const int t_last = min(p_last, seq.length - seq.queries + (row0 + tile * 128 + 127) / a.group);
        float factor = a.scale_log2;
        {
            const char *src = a.q + (seq.first_query + query) * a.q_token_stride + (head * a.group + row % a.group) * a.q_head_stride;
            float down = 1.0f;
            if (BF16) {
                // times a power of two, so that the largest is in [1, 2): exact, but for numbers below 2^-14 of it, which
                // are off by 2^-25 of it at most
                float top = 0.0f;
                if (live)
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(src + i * 16);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u))));
                    }
                const int ex = min(max((__float_as_int(top) >> 23) & 0xff, 8), 246);
                down = __int_as_float((254 - ex) << 23);
                factor *= __int_as_float(ex << 23);
            }
            // a negative scale turns the queries round, so that maxima of scores are maxima of products
            const uint32_t flip = factor < 0.0f ? 0x80008000u : 0u;
            factor = fmaxf(fabsf(factor), 1e-30f);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                uint32_t q[32];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 v = live ? *reinterpret_cast<const uint4 *>(src + c * 128 + i * 16) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        q[4 * i + k] = flip ^ (BF16 ? h2(__floats2half2_rn(__uint_as_float(w[k] << 16) * down, __uint_as_float(w[k] & 0xffff0000u) * down)) : w[k]);
                }
                tmem_st_32x32b_x32(tmem + lanes + P::T_Q + tile * (D / 2) + c * 32, q);
            }
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P::Q_FULL));
        }

        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const int buffer = TILES == 2 ? tile : j & 1, turn = TILES == 2 ? j : j / 2;
            if (!mbar_wait_warp(bar(P::S_FULL + buffer), (uint32_t)(turn & 1), s_abort)) { ok = false; break; }
            tcgen05_fence_after();
            const uint32_t ts = tmem + lanes + P::T_S + buffer * PR_KEYS;
            uint32_t s0[32], s1[32];
            tmem_ld_32x32b_x32(ts, s0);
            tmem_ld_32x32b_x32(ts + 32, s1);
            tmem_ld_wait();
            const int token0 = walk.tile(j0 + j) * PR_KEYS;
            const uint32_t absent = info[j % 16];
            if (absent || token0 + PR_KEYS - 1 > t_first || (a.window && token0 <= t_last - a.window && token0 + PR_KEYS > a.sinks)) {
#pragma unroll
                for (int i = 0; i < PR_KEYS; ++i) {
                    const int token = token0 + i;
                    const bool hidden = token > place || (a.window && token <= place - a.window && token >= a.sinks) || ((absent >> (i / KV_SLAB)) & 1);
                    if (hidden) (i < 32 ? s0[i % 32] : s1[i % 32]) = 0xff800000u;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, fmaxf(__uint_as_float(s0[i]), __uint_as_float(s1[i])));
            top *= factor;
            bool settled = TILES == 2 || j == 0;   // whether the product in front has been seen to end
            if (__any_sync(0xffffffffu, top > m + KV_HEADROOM)) {
                const float now = fmaxf(m, top), shrink = m == -INFINITY ? 0.0f : exp2_fast(m - now);
                m = now;
                l *= shrink;
                if (j > 0) {     // what there is of O shrinks
                    // (two row tiles: S of this tile came behind the product into O)
                    if (TILES == 1 && !mbar_wait_warp(bar(P::O_DONE), (uint32_t)((j - 1) & 1), s_abort)) { ok = false; break; }
                    settled = true;
                    tcgen05_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(tmem + lanes + tile * D + c * 32, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                        tmem_st_32x32b_x32(tmem + lanes + tile * D + c * 32, o);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : KV_SHIFT - m;
            float sum = 0.0f;
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float x = exp2_fast(fmaf(__uint_as_float(i < 16 ? s0[2 * i] : s1[2 * i - 32]), factor, ref));
                const float y = exp2_fast(fmaf(__uint_as_float(i < 16 ? s0[2 * i + 1] : s1[2 * i - 31]), factor, ref));
                sum += x + y;
                p[i] = h2(__floats2half2_rn(x, y));
            }
            l += sum;
            // (every phase is waited for: its parity would not tell the one after the next from it)
            if (!settled && !mbar_wait_warp(bar(P::O_DONE), (uint32_t)((j - 1) & 1), s_abort)) { ok = false; break; }
            tmem_st_32x32b_x32(ts, p);
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P::P_FULL + buffer));
        }
        // ------------------------------ output ------------------------------
        if (ok && tiles) ok = mbar_wait_warp(bar(P::O_DONE), TILES == 2 ? 0u : (uint32_t)((tiles - 1) & 1), s_abort);
        if (!ok) *s_abort = 1;
        if (__all_sync(0xffffffffu, ok)) {
            tcgen05_fence_after();
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            char *dst = live ? out_row(a, seq, head, row, D) : nullptr;
            // (a split leaves maximum, sum and output of each row)
            float *part = a.partial + ((((int64_t)blockIdx.z * a.kv_heads + head) * gridDim.x + row0 / P::ROWS) * P::ROWS + in_block) * (D + 4);
            if (splits > 1 && live) *reinterpret_cast<float2 *>(part) = make_float2(m, l);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (tiles) {
                    tmem_ld_32x32b_x32(tmem + lanes + tile * D + c * 32, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                auto at = [&](int ch) { return __uint_as_float(o[8 * (ch % 4) + ch / 4]); };   // channel 32 c + ch
                if (!live) continue;
                if (splits > 1) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(part + 4 + c * 32 + 4 * i) = make_float4(at(4 * i), at(4 * i + 1), at(4 * i + 2), at(4 * i + 3));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 x = pack4<BF16>(at(8 * i) * inv, at(8 * i + 1) * inv, at(8 * i + 2) * inv, at(8 * i + 3) * inv);
                        const uint2 y = pack4<BF16>(at(8 * i + 4) * inv, at(8 * i + 5) * inv, at(8 * i + 6) * inv, at(8 * i + 7) * inv);
                        *reinterpret_cast<uint4 *>(dst + (c * 32 + 8 * i) * 2) = make_uint4(x.x, x.y, y.x, y.y);
                    }
                }
            }
        }
        tcgen05_fence_before();
    }

    __syncthreads();
    if (*s_abort) {
        // a wait ran out somewhere: no copy may land, and no MMA run, once this CTA has gone
        if (warp == PR_LOAD && lane == 0)
            for (int i = max(0, issued - RS); i < issued; ++i) mbar_wait<100>(bar(P::RAW_FULL + i % RS), (uint32_t)((i / RS) & 1));
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
    plan.splits = 1;
    plan.bytes = 0;
    return plan;
}

template <int D, bool BF16>
int launch(const Attention &a, const PromptPlan &plan, cudaStream_t stream) {
    using P = Prompt<D>;
    auto *kernel = kv_prompt_kernel<D, BF16>;
    int e = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::TOTAL), "atlas_kv_attention");
    if (e != ATLAS_OK) return e;
    kernel<<<dim3((unsigned)plan.blocks, (unsigned)a.kv_heads, (unsigned)(a.batch * plan.splits)), PR_THREADS, P::TOTAL, stream>>>(a, plan.splits);
    e = check_cuda(cudaGetLastError(), "atlas_kv_attention");
    if (e != ATLAS_OK || plan.splits == 1) return e;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(plan.blocks * P::ROWS * (D / 4) / 256), (unsigned)a.kv_heads, (unsigned)a.batch);
    config.blockDim = dim3(256);
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&config, kv_prompt_join_kernel<D, BF16>, a, plan.splits, (int)plan.blocks), "atlas_kv_attention");
}

}  // namespace

bool kv_prompt_serves(const AtlasKvAttention &p) { return p.max_queries * (p.q_heads / p.kv_heads) > 64 && p.batch <= 65535; }

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
