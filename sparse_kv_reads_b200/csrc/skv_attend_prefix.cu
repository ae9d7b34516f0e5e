// Attention of one new token per sequence over a prefix that all sequences share (its cache rows exist once) and over
// each sequence's own rows behind it.
//
// bf16, two launches.  The first reads the prefix once per KV head for all sequences together: their batch x G query rows
// are the M side of tcgen05 products over 128-key tiles (prefix_mma_kernel).  The second attends over the own rows and merges
// everything (prefix_own_kernel); where the prefix is short or the batch small it takes the prefix's rows as well and is the
// only launch.
// float32: a (sequence, KV head) pair walks the prefix and its own rows as one list, half a warp per row, float32
// arithmetic on the CUDA cores.
#include <cuda.h>

#include "skv_attend_finish.cuh"
#include "skv_tcgen05.cuh"

namespace skv {

struct PrefixParams {
    const void *q, *kp, *vp, *k, *v;
    const int32_t *n_dev;
    void *out;
    float *part;       // [batch * h_kv, splits, G, 132]: the prefix's partials, then the own rows'
    int32_t *ticket;   // [batch * h_kv]
    int32_t *status;
    int batch, h_kv, G, n_group, prefix, rows_limit, splits;
    int prefix_splits, own_splits;      // bf16: prefix_splits + own_splits <= splits
    int own_ctas;                       // bf16: CTAs of the second launch per sequence and KV head
    int listed;                         // bf16: rows of the prefix that the second launch reads itself
    int64_t kph, kpr, vph, vpr, ksh, ksr, vsh, vsr;
    float scale_log2;
};

// A key that is no number leaves its head without one, as the definition has it.
__device__ __forceinline__ float quotient(const PrefixParams &, float num, float den) { return den == 0.f ? 0.f : num / den; }

// Own rows of (sequence, KV head) `head`: its length, within the rows the cache has (a longer one is recorded).
__device__ __forceinline__ int own_rows(const PrefixParams &p, int head) {
    const int n = positions_of(p.n_dev, p.n_group, head);
    if (n > p.rows_limit && p.status && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status + head, SKV_ST_BAD_INDEX);
    return min(max(n, 0), p.rows_limit);
}

template <int GP>
__global__ void __launch_bounds__(128) attend_prefix_simple_kernel(const PrefixParams p) {
    constexpr int WARPS = 4;
    __shared__ __align__(16) float red[2 * WARPS * GP * 132];
    __shared__ int s_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y, split = blockIdx.x, h = head % p.h_kv;
    const int G = p.G;
    const int n = p.prefix + own_rows(p, head);
    const int tiles = (n + TILE_ROWS - 1) / TILE_ROWS;
    const int s_eff = min(p.splits, max(1, (tiles + WARPS - 1) / WARPS));
    if (split >= s_eff) return;
    const int slots = s_eff * WARPS, per = (tiles + slots - 1) / slots;
    const int t0 = min((split * WARPS + warp) * per, tiles), t1 = min(t0 + per, tiles);
    const int sub = lane & 15, half = lane >> 4;
    const unsigned hmask = half ? 0xffff0000u : 0x0000ffffu;
    const float *q = static_cast<const float *>(p.q) + (int64_t)head * G * HEAD_DIM;

    float qr[GP][8], acc[GP][8], m[GP], l[GP];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
        m[g] = NEG_BIG;
        l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[g][i] = qr[g][i] = 0.f;
        if (g < G) load8(q + g * HEAD_DIM + sub * 8, qr[g]);
    }
    const int r1 = min(t1 * TILE_ROWS, n);
    for (int r = t0 * TILE_ROWS + half; r < r1; r += 2) {
        const bool shared = r < p.prefix;
        const int64_t own = r - p.prefix;
        const float *kr = shared ? static_cast<const float *>(p.kp) + h * p.kph + (int64_t)r * p.kpr
                             : static_cast<const float *>(p.k) + head * p.ksh + own * p.ksr;
        const float *vr = shared ? static_cast<const float *>(p.vp) + h * p.vph + (int64_t)r * p.vpr
                             : static_cast<const float *>(p.v) + head * p.vsh + own * p.vsr;
        float kv[8], vv[8];
        load8(kr + sub * 8, kv);
        load8(vr + sub * 8, vv);
#pragma unroll
        for (int g = 0; g < GP; ++g) {
            float z = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) z = fmaf(qr[g][e], kv[e], z);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) z += __shfl_xor_sync(hmask, z, o, 16);
            z *= p.scale_log2;
            const float mn = fmaxf(m[g], z);
            const float al = exp2f(m[g] - mn), pr = exp2f(z - mn);
            m[g] = mn;
            l[g] = l[g] * al + pr;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[g][e] = fmaf(pr, vv[e], acc[g][e] * al);
        }
    }
    const int set = warp * 2 + half;
#pragma unroll
    for (int g = 0; g < GP; ++g) {
        if (g >= G) continue;
        float *r = red + (set * G + g) * 132;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[sub * 8 + e] = acc[g][e];
        if (sub == 0) { r[128] = m[g]; r[129] = l[g]; }
    }
    __syncthreads();
    finish_head<float>(p, red, 2 * WARPS, head, split, s_eff, (int64_t)head * p.splits, &s_flag, red, 2 * WARPS * GP);
}

// ---------------------------------------------------------------------------------------------
// The prefix, bf16: rows of all sequences together on the tensor cores
// ---------------------------------------------------------------------------------------------
// A CTA (one per SM) serves one KV head, a run of 128-key tiles and up to 256 query rows.  Two warpgroups of softmax threads
// have an accumulator each (slot 0 and 1): with more than 128 query rows they take 128 rows each of every tile, else both
// have the same rows and take the tiles in turn, and are merged at the end.  A thread owns one row: it reads its 128 scores
// from tensor memory, so that no maximum needs a shuffle, and writes the weights back over them in bf16 as the A operand of
// the second product (which takes A and B of one type, and the values are bf16; half floats would not hold them all, and a
// product with the weights' remainders as well would add a half to those that bound the wide case.  The sum of the weights
// is taken before they are rounded, in float32).  One thread feeds the ring of K and V tiles by TMA (rows beyond the prefix read
// as zeros), one issues
//   S = Q K^T  (both K-major in shared memory)        O += P V  (P in tensor memory, V MN-major)
// with the two slots strictly in turn, so that one's products run beside the other's softmax.  Accumulators are rescaled only
// when a row's maximum rises by more than 8 (base 2).
// What bounds it.  Up to 128 rows the memory: a tile of 64 KB takes an SM about 2,700 cycles, which is the copy rate over 144
// SMs; the rest of 27 us for 8 heads x 32,768 keys (floor 20.5 us) is the start (4,000 cycles to the first scores) and the way
// out.  With more rows the one sequence of products: for each slot of a tile about 560 cycles for the weighted values, 650 for
// the scores (both operands from shared memory, beside the incoming tiles) and 500 of waits and commits between them, 3,430
// cycles a tile where the tensor cores alone need 2,048; a slot's weights lie ready 360 cycles before their turn comes (its
// softmax takes 1,650: loads 115, maximum 280, exponentials 1,230; taken with scale and difference in one fused operation).
// Measured and not kept (128 sequences x 4 query heads x 16,383 keys, 53.5 us with the second launch, as it then was): scores and
// weights by halves of a tile (71.6 us: with 64 keys on N the queries are read from shared memory twice as often), an issuing thread per
// slot (62.4 us: the slots fall into step), weights released by halves (54.9 us).  Within 1 us of it, either way, since the
// softmax does not bound it: half the weights against the standing reference while the maximum is found, products issued by
// a converged warp, barriers looked at ahead of their turn (this one 2.5 us slower for 32 sequences x 32,768 keys); 1 to 5 us
// slower: an eighth to a half of the exponentials by a polynomial on the multiply-add pipe.
constexpr int PT = 128;                                   // keys of a tile, rows of a slot
constexpr int PSTAGES = 2;
constexpr uint32_t P_TILE = PT * 256;                     // bytes of a 128 x 128 bf16 tile: two halves of 64 components
constexpr uint32_t P_OUT = PT * PART_LD * 4;              // bytes of a slot's float32 rows on their way out
constexpr uint32_t P_SMEM = 2 * P_TILE + PSTAGES * 2 * P_TILE + 1024;
static_assert(2 * P_OUT <= 2 * P_TILE + PSTAGES * 2 * P_TILE, "the rows on their way out lie over the tiles");

struct PrefixBars {
    uint64_t kfull[PSTAGES], vfull[PSTAGES], kempty[PSTAGES], vempty[PSTAGES];
    uint64_t sfull[2], pfull[2], done[2], drain;
};

// 384 threads at 168 registers: the softmax warpgroups take 232 each, the third (tiles, products, two idle warps) keeps 40:
// 128 x (2 x 232 + 40) = 384 x 168.
constexpr int P_THREADS = 384;

__global__ void __launch_bounds__(P_THREADS, 1)
prefix_mma_kernel(const PrefixParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ unsigned char raw[];
    __shared__ PrefixBars bars;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_fail;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char *const smem = raw + (base - smem_u32(raw));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, h = blockIdx.z;
    const int rows = p.batch * p.G, row0 = blockIdx.y * 2 * PT;
    const bool both = rows - row0 <= PT;                  // one set of rows: the slots take the tiles in turn
    const int tiles = (p.prefix + PT - 1) / PT;
    const int t0 = (int)((int64_t)tiles * split / p.prefix_splits), t1 = (int)((int64_t)tiles * (split + 1) / p.prefix_splits);
    const int n = t1 - t0;
    const uint32_t kbase = base + 2 * P_TILE;
    const uint32_t b_kfull = smem_u32(bars.kfull), b_vfull = smem_u32(bars.vfull), b_kempty = smem_u32(bars.kempty),
                   b_vempty = smem_u32(bars.vempty), b_sfull = smem_u32(bars.sfull), b_pfull = smem_u32(bars.pfull),
                   b_done = smem_u32(bars.done), b_drain = smem_u32(&bars.drain);
    // one tile's K or V, two boxes of 64 components
    auto load = [&](const CUtensorMap &map, uint32_t dst, uint32_t bar, int tile) {
        mbar_expect(bar, P_TILE);
        tma_load_3d(dst, &map, bar, 0, tile * PT, h);
        tma_load_3d(dst + P_TILE / 2, &map, bar, 64, tile * PT, h);
    };
    if (tid == 256) {
        for (int i = 0; i < PSTAGES; ++i) {
            mbar_init(b_kfull + 8 * i, 1); mbar_init(b_vfull + 8 * i, 1);
            mbar_init(b_kempty + 8 * i, 1); mbar_init(b_vempty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_sfull + 8 * i, 1); mbar_init(b_pfull + 8 * i, PT / 32); mbar_init(b_done + 8 * i, 1);
        }
        mbar_init(b_drain, 1);
        s_fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_proxy();
    }
    pdl_wait();
    pdl_trigger();
    // Queries into the 128-byte swizzle, 16 bytes at a time; rows beyond the last are zero.  A negative softmax scale goes
    // into their sign: the running maximum is one of scaled scores.  All of a thread's loads are requested at once, and ahead
    // of the other tiles: behind them they took up to 14,000 cycles.
    {
        constexpr int CHUNKS = (2 * PT * 16 + P_THREADS - 1) / P_THREADS;
        const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
        const int qrows = both ? PT : 2 * PT;
        uint4 v[CHUNKS];
#pragma unroll
        for (int e = 0; e < CHUNKS; ++e) {
            const int i = tid + e * P_THREADS, row = row0 + (i >> 4);
            v[e] = make_uint4(0u, 0u, 0u, 0u);
            if ((i >> 4) < qrows && row < rows) {
                const int b = (int)((unsigned)row / (unsigned)p.G), g = row - b * p.G;
                v[e] = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p.q) +
                                                        (((int64_t)b * p.h_kv + h) * p.G + g) * HEAD_DIM + (i & 15) * 8);
            }
        }
        if (tid == 256) {
            for (int i = 0; i < min(n, PSTAGES); ++i) {
                load(kmap, kbase + i * 2 * P_TILE, b_kfull + 8 * i, t0 + i);
                load(vmap, kbase + i * 2 * P_TILE + P_TILE, b_vfull + 8 * i, t0 + i);
            }
        }
        // Only behind the wait: an allocation blocks without a limit, so a launch that has started early must not hold the
        // columns that a launch ahead of it has still to ask for.
        if (warp == 9) {
            __syncwarp();                                 // (its lanes may have parted at the last row)
            tmem_alloc(smem_u32(&s_tmem), 512);
        }
#pragma unroll
        for (int e = 0; e < CHUNKS; ++e) {
            const int i = tid + e * P_THREADS, r = i >> 4, c = i & 15, rr = r & (PT - 1);
            if (r >= qrows) continue;
            v[e].x ^= flip; v[e].y ^= flip; v[e].z ^= flip; v[e].w ^= flip;
            unsigned char *to = smem + (r >> 7) * P_TILE + (c >> 3) * (P_TILE / 2) + rr * 128;
            *reinterpret_cast<uint4 *>(to + (((c & 7) ^ (rr & 7)) << 4)) = v[e];
        }
    }
    fence_async_proxy();
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = s_tmem;

    if (warp >= 8) {
        fewer_registers<40>();
        if (warp == 8) {
            // ---- tiles, by TMA ----
            if (lane == 0) {
                int i = min(n, PSTAGES);
                bool ok = true;
                for (; i < n; ++i) {
                    const int s = i % PSTAGES;
                    const uint32_t kt = kbase + s * 2 * P_TILE, turn = (i / PSTAGES - 1) & 1;
                    if (!(ok = mbar_wait(b_kempty + 8 * s, turn))) break;
                    load(kmap, kt, b_kfull + 8 * s, t0 + i);
                    if (!(ok = mbar_wait(b_vempty + 8 * s, turn))) {
                        mbar_wait(b_kfull + 8 * s, (i / PSTAGES) & 1);
                        break;
                    }
                    load(vmap, kt + P_TILE, b_vfull + 8 * s, t0 + i);
                }
                if (!ok) s_fail = 1;
                for (int j = max(0, i - PSTAGES); j < i; ++j) {            // no copy is in flight when the CTA ends
                    mbar_wait(b_kfull + 8 * (j % PSTAGES), (j / PSTAGES) & 1);
                    mbar_wait(b_vfull + 8 * (j % PSTAGES), (j / PSTAGES) & 1);
                }
            }
        } else if (warp == 9) {
            // ---- products ----
            if (lane == 0) {
                constexpr uint32_t ID_S = idesc_bf16(PT, PT, false), ID_O = idesc_bf16(PT, HEAD_DIM, true);
                bool ok = true;
                // slot w's scores of tile i; `free_k`: nothing reads the key tile afterwards
                auto scores = [&](int i, int w, bool free_k) {
                    const int s = i % PSTAGES;
                    if (!ok || !(ok = mbar_wait(b_kfull + 8 * s, (i / PSTAGES) & 1))) return;
                    tcgen05_after_sync();
                    const uint32_t qt = base + (both ? 0 : w) * P_TILE, kt = kbase + s * 2 * P_TILE;
    #pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t at = (k >> 2) * (P_TILE / 2) + (k & 3) * 32;
                        mma_ss(tmem + w * PT, smem_desc(qt + at, 1024), smem_desc(kt + at, 1024), ID_S, k > 0);
                    }
                    tcgen05_commit(b_sfull + 8 * w);
                    if (free_k) tcgen05_commit(b_kempty + 8 * s);
                };
                // slot w's weighted values of tile i, its turn number j
                auto values = [&](int i, int w, int j, bool free_v, bool last) {
                    const int s = i % PSTAGES;
                    if (!ok || !(ok = mbar_wait(b_pfull + 8 * w, j & 1)) || !(ok = mbar_wait(b_vfull + 8 * s, (i / PSTAGES) & 1)))
                        return;
                    tcgen05_after_sync();
                    const uint32_t vt = kbase + s * 2 * P_TILE + P_TILE;
    #pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_ts(tmem + 256 + w * PT, tmem + w * PT + k * 8, smem_desc(vt + k * 2048, 1024, P_TILE / 2), ID_O,
                               j > 0 || k > 0);
                    if (free_v) tcgen05_commit(b_vempty + 8 * s);
                    if (last) tcgen05_commit(b_done + 8 * w);
                };
                if (both) {
                    scores(0, 0, true);
                    if (n > 1) scores(1, 1, true);
                    for (int i = 0; i < n; ++i) {
                        values(i, i & 1, i >> 1, true, i + 2 >= n);
                        if (i + 2 < n) scores(i + 2, i & 1, true);
                    }
                } else {
                    scores(0, 0, false);
                    scores(0, 1, true);
                    for (int i = 0; i < n; ++i)
                        for (int w = 0; w < 2; ++w) {
                            values(i, w, i, w == 1, i + 1 == n);
                            if (i + 1 < n) scores(i + 1, w, w == 1);
                        }
                }
                if (!ok) s_fail = 1;
                tcgen05_commit(b_drain);                      // no product is in flight when the CTA ends
                mbar_wait(b_drain, 0);
            }
        }
    } else {
        // ---- softmax: one row per thread ----
        more_registers<232>();
        const int w = warp >> 2, r = tid & (PT - 1);
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);        // this warp's 32 lanes
        const uint32_t sc = mine + w * PT, oc = mine + 256 + w * PT;
        const float scale = fabsf(p.scale_log2);
        const int turns = both ? (n - w + 1) / 2 : n;
        float m = NEG_BIG, l = 0.f;                           // the row's reference (a score before the scale) and sum of weights
        bool ok = true;
        for (int j = 0; j < turns; ++j) {
            const int i = both ? 2 * j + w : j;
            if (!(ok = mbar_wait_warp(b_sfull + 8 * w, j & 1))) break;
            tcgen05_after_sync();
            uint32_t x[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(sc + c * 32, x[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld_done(x[c]);
            const int left = p.prefix - (t0 + i) * PT;    // keys of this tile
            if (left < PT) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (c * 32 + e >= left) x[c][e] = 0xff800000u;
            }
            float top[4] = {NEG_BIG, NEG_BIG, NEG_BIG, NEG_BIG};
#pragma unroll
            for (int e = 0; e < 32; e += 2)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    top[c] = fmaxf(fmaxf(top[c], __uint_as_float(x[c][e])), __uint_as_float(x[c][e + 1]));
            const float z = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (__any_sync(0xffffffffu, (z - m) * scale > 8.f)) {
                const float nm = fmaxf(m, z), al = fast_exp2((m - nm) * scale);
                m = nm;
                l *= al;
                if (j > 0) {                              // (the products up to the tile before have ended: S came after them)
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        uint32_t o[16];
                        tmem_ld16(oc + c * 16, o);
                        tmem_ld_done(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * al);
                        tmem_st16(oc + c * 16, o);
                    }
                }
            }
            float2 sum[4] = {};
            // Differences first, then the scale: the largest weight is one however large the scores.  (The maximum's rounded
            // product taken off a fused product is up to 2^-25 of it away from that; 54.5 against 54.8 us at 128 sequences.)
            const float2 mul = make_float2(scale, scale), sub = make_float2(-m, -m);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float2 a = mul2(add2(make_float2(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), sub), mul);
                    a.x = fast_exp2(a.x);
                    a.y = fast_exp2(a.y);
                    sum[(e >> 1) & 3] = add2(sum[(e >> 1) & 3], a);
                    pk[e >> 1] = pack_bf16(a.x, a.y);
                }
                tmem_st16(sc + c * 16, pk);               // over scores that are in registers by now
            }
            const float2 all = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
            l += all.x + all.y;
            tcgen05_wait_st();
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_pfull + 8 * w);
        }
        m *= scale;                                           // base 2, as the partials have it
        if (ok && turns > 0) ok = mbar_wait_warp(b_done + 8 * w, 0);
        if (!ok) s_fail = 1;
        // Both slots' products have ended: the tiles' memory is free.  The fences stand on either side of the barrier, since a
        // warp reads the other slot's sums below, whose end only that slot's warps have waited for.
        tcgen05_before_sync();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        tcgen05_after_sync();
        const bool fold = both && n > 1;                  // the two slots have the same rows: a half of the columns each
        float *out = reinterpret_cast<float *>(smem + (fold ? 0 : w) * P_OUT) + r * PART_LD;
        const int row = row0 + (both ? 0 : w * PT) + r, b = (int)((unsigned)row / (unsigned)p.G), g = row - b * p.G;
        float *dst = p.part + ((((int64_t)b * p.h_kv + h) * p.splits + split) * p.G + g) * PART_LD;
        if (fold) {
            float2 *ml = reinterpret_cast<float2 *>(smem + P_OUT);
            ml[w * PT + r] = make_float2(m, l);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float2 a = ml[r], o = ml[PT + r];
            const float M = fmaxf(a.x, o.x), f0 = fast_exp2(a.x - M), f1 = fast_exp2(o.x - M);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t x[32], y[32];
                tmem_ld32(mine + 256 + w * 64 + c * 32, x);
                tmem_ld32(mine + 256 + PT + w * 64 + c * 32, y);
                tmem_ld_done(x);
                tmem_ld_done(y);
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4 *>(out + w * 64 + c * 32 + e) =
                        make_float4(fmaf(f1, __uint_as_float(y[e]), f0 * __uint_as_float(x[e])),
                                    fmaf(f1, __uint_as_float(y[e + 1]), f0 * __uint_as_float(x[e + 1])),
                                    fmaf(f1, __uint_as_float(y[e + 2]), f0 * __uint_as_float(x[e + 2])),
                                    fmaf(f1, __uint_as_float(y[e + 3]), f0 * __uint_as_float(x[e + 3])));
            }
            if (w == 1) *reinterpret_cast<float4 *>(out + HEAD_DIM) = make_float4(M, fmaf(f1, o.y, f0 * a.y), 0.f, 0.f);
            if (row < rows) {
                fence_async_proxy();
                bulk_store(dst + w * 64, smem_u32(out + w * 64), w ? (PART_LD - 64) * 4 : 64 * 4);
            }
        } else if (turns > 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(oc + c * 32, o);
                tmem_ld_done(o);
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<uint4 *>(out + c * 32 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
            *reinterpret_cast<float4 *>(out + HEAD_DIM) = make_float4(m, l, 0.f, 0.f);
            if (row < rows) {
                fence_async_proxy();
                bulk_store(dst, smem_u32(out), PART_LD * 4);
            }
        }
        bulk_store_wait_read();
        tcgen05_before_sync();
    }
    __syncwarp();
    __syncthreads();
    if (s_fail && p.status)
        for (int b = tid; b < p.batch; b += P_THREADS) atomicOr(p.status + b * p.h_kv + h, SKV_ST_WAIT_TIMEOUT);
    if (warp == 9) {
        tcgen05_after_sync();
        tmem_free(tmem, 512);
    }
}

// The sequences' own rows, and everything merged: grid (CTAs, sequence x KV head).  Own rows that one CTA serves alone may be
// served by several all the same, each for some of the query heads: the partials of a long prefix take longer to join than
// a few own rows to read (8 sequences of one KV head with 8 query heads, 30,000 + 100 rows: 32 us with one CTA per head, 17.6
// with eight).  With `listed`, the prefix's rows too, as one list ahead of the own ones (short prefixes and small batches,
// which the second-level cache serves).  Bounded by latencies: 46 MB of own rows and 18 partials each of 512 query rows take
// 10 us alone, 7 us of which the memory needs.
// STAGES tiles of 16 rows per warp: as many as the shared memory allows at the CTAs per SM that the grid makes.  Beyond three
// per SM one tile and four CTAs: more CTAs at once are worth more than tiles asked for ahead (1,024 heads: 49 us against 55 us
// for both launches with 40 own rows, 96 against 95 with 1,000).
template <int STAGES>
__global__ void __launch_bounds__(128, STAGES == 1 ? 4 : 3) prefix_own_kernel(const PrefixParams p) {
    constexpr int WARPS = 4;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t s_vmask[WARPS][STAGES];
    __shared__ int s_flag;
    const int tid = threadIdx.x, warp = tid >> 5, head = blockIdx.y, split = blockIdx.x, h = head % p.h_kv, G = p.G;
    const int n = own_rows(p, head);
    const int shared_tiles = (p.listed + TILE_ROWS - 1) / TILE_ROWS, tiles = shared_tiles + (n + TILE_ROWS - 1) / TILE_ROWS;
    // tiles of a warp at least before another CTA takes part: four where the prefix's partials have to be joined as well
    const int least = WARPS * (p.prefix_splits > 0 ? 4 : 1);
    const int s_eff = min(p.own_splits, max(1, (tiles + least - 1) / least));
    const int joint = s_eff == 1 ? min((int)gridDim.x, G) : 1;         // CTAs that share the query heads
    if (split >= max(s_eff, joint)) {
        pdl_wait();
        return;
    }
    const int slots = s_eff * WARPS, per = (tiles + slots - 1) / slots;
    const int t0 = min((s_eff == 1 ? warp : split * WARPS + warp) * per, tiles), t1 = min(t0 + per, tiles);
    const char *ko = static_cast<const char *>(p.k) + (int64_t)head * p.ksh * 2;
    const char *vo = static_cast<const char *>(p.v) + (int64_t)head * p.vsh * 2;
    WarpAttendT<STAGES> wa;
    wa.init(static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)head * G * HEAD_DIM, G, smem + warp * (STAGES * 8192),
            s_vmask[warp], static_cast<const char *>(p.kp) + (int64_t)h * p.kph * 2,
            static_cast<const char *>(p.vp) + (int64_t)h * p.vph * 2, p.kpr * 2, p.vpr * 2, p.scale_log2);
    if (t0 < shared_tiles) wa.run(t0, min(t1, shared_tiles), [&](int row) { return row < p.listed ? row : -1; });
    wa.Kb = ko; wa.Vb = vo; wa.krow = p.ksr * 2; wa.vrow = p.vsr * 2;
    if (t1 > shared_tiles)
        wa.run(max(t0, shared_tiles) - shared_tiles, t1 - shared_tiles, [&](int row) { return row < n ? row : -1; });
    __syncthreads();
    float *red = reinterpret_cast<float *>(smem);
    wa.store_partial(red, warp, G);
    __syncthreads();
    const int parts = p.prefix_splits + s_eff;
    const int64_t slot0 = (int64_t)head * p.splits;
    pdl_wait();                            // the prefix's partials, and whoever read the output before
    pdl_trigger();
    if (s_eff == 1) {
        // Alone: the prefix's partials straight from where they lie.  Every warp folds a quarter of each row's into its own
        // partial (a lane has four columns; the loads of two query heads are in flight together), then the four are joined.
        constexpr int AT_ONCE = STAGES == 1 ? 3 : 5;
        const int lane = tid & 31;
        const int ga = G * split / joint, gb = G * (split + 1) / joint;      // this CTA's query heads
        for (int g0 = ga; g0 < gb; g0 += 2) {
            float M[2], dn[2];
            float4 nm[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float *r = red + (warp * G + min(g0 + e, gb - 1)) * PART_LD;
                M[e] = r[128]; dn[e] = r[129];
                nm[e] = *reinterpret_cast<const float4 *>(r + lane * 4);
            }
            for (int i0 = warp; i0 < p.prefix_splits; i0 += WARPS * AT_ONCE) {
                float2 ml[2][AT_ONCE];
                float4 a[2][AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        ml[e][i] = make_float2(NEG_BIG, 0.f);
                        a[e][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (i0 + i * WARPS < p.prefix_splits) {
                            const float *r = p.part + ((slot0 + i0 + i * WARPS) * G + min(g0 + e, gb - 1)) * PART_LD;
                            ml[e][i] = __ldcg(reinterpret_cast<const float2 *>(r + 128));
                            a[e][i] = __ldcg(reinterpret_cast<const float4 *>(r + lane * 4));
                        }
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = M[e];
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, ml[e][i].x);
                    const float al = fast_exp2(M[e] - top);
                    M[e] = top;
                    dn[e] *= al;
                    nm[e].x *= al; nm[e].y *= al; nm[e].z *= al; nm[e].w *= al;
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) {
                        const float f = fast_exp2(ml[e][i].x - top);
                        dn[e] = fmaf(f, ml[e][i].y, dn[e]);
                        nm[e].x = fmaf(f, a[e][i].x, nm[e].x); nm[e].y = fmaf(f, a[e][i].y, nm[e].y);
                        nm[e].z = fmaf(f, a[e][i].z, nm[e].z); nm[e].w = fmaf(f, a[e][i].w, nm[e].w);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (g0 + e >= gb) continue;
                float *r = red + (warp * G + g0 + e) * PART_LD;
                __syncwarp();
                *reinterpret_cast<float4 *>(r + lane * 4) = nm[e];
                if (lane == 0) { r[128] = M[e]; r[129] = dn[e]; }
            }
        }
        __syncthreads();
        for (int g = ga; g < gb; ++g) {
            float M = NEG_BIG, dn = 0.f, nm = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) M = fmaxf(M, red[(w * G + g) * PART_LD + 128]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float *r = red + (w * G + g) * PART_LD;
                const float f = fast_exp2(r[128] - M);
                dn += f * r[129];
                nm += f * r[tid];
            }
            store_out(static_cast<__nv_bfloat16 *>(p.out) + ((int64_t)head * G + g) * HEAD_DIM + tid, quotient(p, nm, dn));
        }
        return;
    }
    publish_head<__nv_bfloat16>(p, red, WARPS, head, p.prefix_splits + split, parts, slot0);
    __threadfence();
    __syncthreads();
    if (tid == 0) s_flag = atomicAdd(p.ticket + head, 1) == s_eff - 1;
    __syncthreads();
    if (!s_flag) return;
    __threadfence();
    merge_head<__nv_bfloat16>(p, head, parts, slot0, red, WARPS * STAGES * 8192 / (PART_LD * 4));
}

static int launch_prefix_simple(const PrefixParams &p, cudaStream_t st) {
    const dim3 grid(p.splits, p.batch * p.h_kv);
    if (p.G <= 1) attend_prefix_simple_kernel<1><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 2) attend_prefix_simple_kernel<2><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 4) attend_prefix_simple_kernel<4><<<grid, 128, 0, st>>>(p);
    else attend_prefix_simple_kernel<8><<<grid, 128, 0, st>>>(p);
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

template <int STAGES>
static int launch_own(const PrefixParams &p, cudaStream_t st) {
    constexpr int SMEM = 4 * STAGES * 8192;
    static bool configured[64] = {};       // the attribute is kept per device
    int dev = 0;
    SKV_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return SKV_E_RANGE;
    if (!configured[dev]) {
        SKV_CUDA_OK(cudaFuncSetAttribute(prefix_own_kernel<STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        configured[dev] = true;
    }
    // Behind the prefix's launch, which waits for everything before it, this one may always start early: its own rows are
    // read while the last tiles of the prefix are multiplied.
    SKV_CUDA_OK(launch_as(pdl_allowed() && p.prefix_splits > 0, prefix_own_kernel<STAGES>, dim3(p.own_ctas, p.batch * p.h_kv),
                          dim3(128), SMEM, st, p));
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

// The prefix's rows go through the list where reading them once per sequence moves at most this much, for the most part
// through the second-level cache (two sequences of 8,192 rows, 67 MB: 14.3 us by the list, 16.4 by the tiles; four, 134 MB:
// 21.1 and 15.2; four of 333 rows: 6.7 and 9.5).
constexpr int64_t LIST_BYTES = 64 << 20;

// Most CTAs the prefix of a KV head is split over: one per SM over all heads and row groups.  (A call uses at most a third
// of the prefix's tiles: a partial costs the merge as much as a tile costs its CTA.)
static int prefix_splits_of(int batch, int h_kv, int G) {
    const int groups = (batch * G + 2 * PT - 1) / (2 * PT), s = device_sm_count() / (h_kv * groups);
    return s < 1 ? 1 : s;
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Map of [h_kv, prefix, 128] bf16 rows in boxes of 128 rows x 64 components, 128-byte swizzle; false where the strides or the
// address do not allow one.
static bool prefix_map(CUtensorMap *map, const void *x, int h_kv, int prefix, int64_t head_stride, int64_t row_stride) {
    static EncodeTiled encode = nullptr;
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return false;
        encode = reinterpret_cast<EncodeTiled>(fn);
    }
    if (prefix == 1) row_stride = HEAD_DIM;               // (a stride that no address uses may be anything)
    if (h_kv == 1) head_stride = row_stride;
    if (row_stride < HEAD_DIM || head_stride <= 0) return false;
    const cuuint64_t dims[3] = {HEAD_DIM, (cuuint64_t)prefix, (cuuint64_t)h_kv};
    const cuuint64_t strides[2] = {(cuuint64_t)row_stride * 2, (cuuint64_t)head_stride * 2};
    const cuuint32_t box[3] = {64, PT, 1}, unit[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(x), dims, strides, box, unit,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// CTAs per KV head and 256 query rows of the prefix's own launch, with its maps; 0: the second launch reads the prefix as well.
static int prefix_tile_ctas(const PrefixParams &p, CUtensorMap *kmap, CUtensorMap *vmap) {
    const int heads = p.batch * p.h_kv, tiles = (p.prefix + PT - 1) / PT;
    // (a scale of zero by the list as well: the tiles mark keys beyond the prefix by scores of -inf, which times zero is no number)
    const bool list = (int64_t)heads * p.prefix * 2 * HEAD_DIM * 2 <= LIST_BYTES || p.scale_log2 == 0.f;
    int ps = list ? 0 : prefix_splits_of(p.batch, p.h_kv, p.G);
    if (ps > (tiles + 2) / 3) ps = (tiles + 2) / 3;
    if (ps > p.splits - 1) ps = p.splits - 1;
    if (ps > 0 && (!prefix_map(kmap, p.kp, p.h_kv, p.prefix, p.kph, p.kpr) ||
                   !prefix_map(vmap, p.vp, p.h_kv, p.prefix, p.vph, p.vpr)))
        ps = 0;                            // (strides that no map can have)
    return ps;
}

static int launch_prefix_mma(PrefixParams p, cudaStream_t st) {
    const int heads = p.batch * p.h_kv;
    CUtensorMap kmap, vmap;
    const int ps = prefix_tile_ctas(p, &kmap, &vmap);
    int own = skv_attend_splits(heads);
    if (own > p.splits - ps) own = p.splits - ps;
    p.prefix_splits = ps;
    p.own_splits = own;
    p.listed = ps > 0 ? 0 : p.prefix;
    int joint = 2 * device_sm_count() / heads;             // two CTAs per SM at most share a head's partials out
    joint = joint > p.G ? p.G : joint;
    p.own_ctas = ps > 0 && joint > own ? joint : own;
    if (ps > 0) {
        static bool configured[64] = {};   // the attribute is kept per device
        int dev = 0;
        SKV_CUDA_OK(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64) return SKV_E_RANGE;
        if (!configured[dev]) {
            SKV_CUDA_OK(cudaFuncSetAttribute(prefix_mma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM));
            configured[dev] = true;
        }
        const int groups = (p.batch * p.G + 2 * PT - 1) / (2 * PT);
        SKV_CUDA_OK(launch_early(prefix_mma_kernel, dim3(ps, groups, p.h_kv), dim3(P_THREADS), P_SMEM, st, p, kmap, vmap));
    }
    const int ctas = heads * p.own_ctas, sms = device_sm_count();
    return ctas <= sms ? launch_own<6>(p, st) : ctas <= 2 * sms ? launch_own<3>(p, st) : ctas <= 3 * sms ? launch_own<2>(p, st) : launch_own<1>(p, st);
}

}  // namespace skv

using namespace skv;

extern "C" int skv_prefix_splits(int batch, int h_kv, int G, int dtype) {
    if (batch <= 0 || h_kv <= 0 || (int64_t)batch * h_kv > 65535) return SKV_E_RANGE;
    if (G < 1 || G > 8) return SKV_E_DIM;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    const int own = skv_attend_splits(batch * h_kv);
    return dtype == SKV_F32 ? own : own + prefix_splits_of(batch, h_kv, G);
}

extern "C" int64_t skv_prefix_workspace_bytes(int batch, int h_kv, int G, int d, int splits) {
    if (batch <= 0 || h_kv <= 0) return SKV_E_RANGE;
    return skv_attend_workspace_bytes(batch * h_kv, G, d, splits);
}

// The caches of a call into the kernels' parameters, checked.
static int prefix_check(const skv_prefix *c, int splits, float scale, PrefixParams &p) {
    if (!c) return SKV_E_NULL;
    if ((c->prefix > 0 && (!c->k_prefix || !c->v_prefix)) || (c->rows_limit > 0 && (!c->k || !c->v))) return SKV_E_NULL;
    if (c->d != HEAD_DIM) return SKV_E_DIM;
    if (c->dtype != SKV_BF16 && c->dtype != SKV_F32) return SKV_E_DTYPE;
    if (c->G < 1 || c->G > 8) return SKV_E_DIM;
    if (c->batch <= 0 || c->h_kv <= 0 || (int64_t)c->batch * c->h_kv > 65535 || c->prefix < 0 || c->rows_limit < 0 ||
        (int64_t)c->prefix + c->rows_limit > 0x7fffffff - 64 || splits <= 0 || splits > 65535 || c->n_group < 0)
        return SKV_E_RANGE;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_prefix) || !aligned16(c->v_prefix)) return SKV_E_ALIGN;
    const int per16 = c->dtype == SKV_BF16 ? 8 : 4;
    const int64_t strides[8] = {c->kp_head_stride, c->kp_row_stride, c->vp_head_stride, c->vp_row_stride,
                                c->k_head_stride, c->k_row_stride, c->v_head_stride, c->v_row_stride};
    for (int i = 0; i < 8; ++i) {
        const int rows = i < 4 ? c->prefix : c->rows_limit;
        if (strides[i] % per16 || ((i & 1) && rows > 1 && strides[i] < HEAD_DIM)) return SKV_E_ALIGN;
    }
    p.kp = c->k_prefix; p.vp = c->v_prefix; p.k = c->k; p.v = c->v;
    p.batch = c->batch; p.h_kv = c->h_kv; p.G = c->G; p.n_group = c->n_group; p.prefix = c->prefix; p.rows_limit = c->rows_limit;
    p.splits = splits;
    p.kph = c->kp_head_stride; p.kpr = c->kp_row_stride; p.vph = c->vp_head_stride; p.vpr = c->vp_row_stride;
    p.ksh = c->k_head_stride; p.ksr = c->k_row_stride; p.vsh = c->v_head_stride; p.vsr = c->v_row_stride;
    p.scale_log2 = scale * LOG2E;
    return SKV_OK;
}

extern "C" int skv_prefix_launches(const skv_prefix *c, int splits, float scale) {
    PrefixParams p = {};
    const int rc = prefix_check(c, splits, scale, p);
    if (rc) return rc;
    CUtensorMap kmap, vmap;
    return c->dtype == SKV_BF16 && prefix_tile_ctas(p, &kmap, &vmap) > 0 ? 2 : 1;
}

extern "C" int skv_attend_prefix(const skv_prefix *c, const void *q, const int32_t *n_dev, void *out, void *workspace, int splits,
                                 int32_t *status, float scale, void *stream) {
    if (!q || !n_dev || !out || !workspace) return SKV_E_NULL;
    PrefixParams p = {};
    const int rc = prefix_check(c, splits, scale, p);
    if (rc) return rc;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return SKV_E_ALIGN;
    p.q = q; p.n_dev = n_dev; p.out = out; p.status = status;
    p.part = static_cast<float *>(workspace);
    p.ticket = reinterpret_cast<int32_t *>(p.part + (int64_t)c->batch * c->h_kv * splits * c->G * PART_LD);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->dtype == SKV_F32) return launch_prefix_simple(p, st);
    return launch_prefix_mma(p, st);
}
