// Attention of one new token per sequence over a quantised KV cache, split over CTAs, merged by the last CTA of a head.
//
// bf16 queries: tensor-core kernel.  Both products take half-float operands, because a code turns into a half float with
// one byte permutation or one logic operation: 0x6400 | c is 1024 + c, 0x6400 | c << 4 is 1024 + 16 c.
//   S^T = K Q^T (16 keys on M, up to 8 query heads on N).  The order of the 128 components is free as long as both sides
//     agree on it, so a lane takes a row's bytes 16 at a time and the queries are fetched in the matching order.  The
//     offsets (1152 = 1024 + 128 in 8 bits) stay in the codes: the accumulators start at minus the offset times the sum of
//     the query.  Queries are scaled by a power of two to a largest component in [1, 2), which half floats hold to 2^-25 of
//     that (4 bits: 2^-21 in odd places, whose codes lie four bits higher).  Scores of up to 2^104 come out right whatever the
//     sizes of queries and keys.
//   O^T = V^T (P vs): component d of the values on M, keys on K.  A lane reads the same bytes of the value rows of its
//     four keys and pairs them up by permutation.  The value's scale goes into the weights (per scale group in 4 bits).
// A warp has a ring of tiles of its own in shared memory, filled by 16-byte asynchronous copies and laid out so that neither
// the rows' nor the columns' reads meet in a bank.  (Loads straight into registers kept one tile in flight per warp: 109 us
// against 92 us for 64 heads of 32,768 8-bit rows, 85 against 75 us in 4 bits.)
// What bounds it: 8 bits, the memory (64 heads of 32,768 rows: 83 us at the measured copy rate); 4 bits, the instructions
// that turn two codes a byte into fragments (325 per 16 rows; the integer pipe is 53 % busy, the memory 60 %).
// A reference for each value group costs 5 of them (75.4 against 74.2 us with one for all four, which held a group 2^-16 of the
// largest to 5e-4 only).
// Running references per head, in base 2: m for the sum of weights (largest score) and, for each scale group of the values, r for
// the group's accumulators (largest score + log2 of the value's scale), so that the half floats 2^(z - r) vs keep their
// precision whatever the scales of rows and groups (of weights down to 2^-126 of the head's largest).  m is only raised when
// a score passes it by 8, r when a half float passes 2^15 (to 2^4 then), so that most tiles need no shuffles.
// A weight is rounded to 11 bits; sums and accumulators are float32.
// float32 queries: half a warp per row, float32 arithmetic on the CUDA cores.
#include <cuda_fp16.h>

#include "skv_attend_finish.cuh"
#include "skv_quant.cuh"

namespace skv {

struct AttendQuantParams {
    const void *q;
    const unsigned char *kc, *vc;
    const __nv_bfloat16 *scale;
    const int32_t *n_dev;
    void *out;
    float *part;       // [ctas + heads, G, 132]
    int32_t *ticket;   // [heads]
    int heads, G, n_group, capacity;
    int ctas;          // CTAs that share the rows
    int splits;        // CTAs per head of the float32 kernel
    int rows;          // rows of 132 floats of shared memory
    float scale_log2;
};

// A key without a number (NaN scale) leaves its head without one, as the definition has it.
__device__ __forceinline__ float quotient(const AttendQuantParams &, float num, float den) { return den == 0.f ? 0.f : num / den; }

template <int BITS, int GP>
__global__ void __launch_bounds__(128) attend_quant_simple_kernel(const AttendQuantParams p) {
    using Q = Quant<BITS>;
    constexpr int WARPS = 4;
    __shared__ __align__(16) float red[2 * WARPS * GP * 132];
    __shared__ int s_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y, split = blockIdx.x;
    const int G = p.G;
    const int n = min(max(positions_of(p.n_dev, p.n_group, head), 0), p.capacity);
    // 16-row tiles in contiguous runs over the head's (splits x warps), as in the list-driven attention
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
        const int64_t row = (int64_t)head * p.capacity + r;
        const __nv_bfloat16 *s = p.scale + row * Q::SCALES + group_of<BITS>(sub);
        float kv[8], vv[8];
        restore_row8<BITS>(p.kc + row * Q::ROW_BYTES, sub, __bfloat162float(s[0]), kv);
        restore_row8<BITS>(p.vc + row * Q::ROW_BYTES, sub, __bfloat162float(s[Q::GROUPS]), vv);
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
// tensor-core path
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}
__device__ __forceinline__ uint32_t hsub(uint32_t x, float by) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&x), __float2half2_rn(by));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t hfma(uint32_t x, float mul, float add) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&x), __float2half2_rn(mul), __float2half2_rn(add));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// the larger magnitudes of two pairs (NaN where both have none)
__device__ __forceinline__ uint32_t hmax(uint32_t x, uint32_t y) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2 *>(&x), __habs2(*reinterpret_cast<const __half2 *>(&y)));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ float bf16_low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
constexpr uint32_t F16_1024 = 0x64006400u;                // two half floats of 1024, whose last place counts 1

// d = a b + c: the start of a chain of products (d and c apart, so that c need not be copied first)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// log2 of a scale: zero or a normal number (-inf for zero)
__device__ __forceinline__ float log2_scale(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What one lane holds of 16 cached positions: lane = 4 g + t.  Keys: rows g and g + 8; values: rows 2t, 2t+1, 2t+8, 2t+9.
template <int BITS>
struct RawTile;
template <>
struct RawTile<8> {
    uint4 k[2][2];                                        // [row g, g + 8][16-byte chunk 2t, 2t + 1]
    uint4 v[4];                                           // chunk g of the four rows
    uint32_t s[2];                                        // (key scale, value scale) of rows g, g + 8
};
template <>
struct RawTile<4> {
    uint4 k[2];                                           // chunk t: runs 2t and 2t + 1 of every scale group
    uint2 v[4];                                           // bytes 8g .. 8g+7: run g of every scale group
    uint4 s[2];                                           // four key scales, four value scales
};

template <int BITS>
struct WarpAttendQuant {
    using Q = Quant<BITS>;
    static constexpr int GR = Q::GROUPS;
    uint32_t qb[8][2];                 // Q^T fragments in the order of the codes, column = head g
    float off[GR][2];                  // what the accumulators of heads 2t, 2t + 1 start from, per scale group
    float acc[8][4];                   // O^T: 8-bit tile j: components 16 g + 2 j and the next; 4-bit tile (group, i): 32 group
                                       // + 4 g + 2 i and the next
    float mA, mB, lA, lB;              // reference of the weights / partial sum of heads 2t, 2t + 1
    float rA[GR], rB[GR], fA[GR], fB[GR];                    // reference of each scale group's accumulators, and 2^(m - r)
    float qsA, qsB;                    // score scale of the two heads, with the query's power of two
    int g, t;

    __device__ __forceinline__ void init(const __nv_bfloat16 *q, int G, float scale_log2) {
        const int lane = threadIdx.x & 31;
        g = lane >> 2; t = lane & 3;
        // component index of the eight 4-component runs this lane owns of head g's query
        float x[8][4];
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const int d = BITS == 8 ? 32 * t + 4 * s : 32 * (s >> 1) + 8 * t + 4 * (s & 1);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (g < G) v = load4(q + g * HEAD_DIM + d);
            x[s][0] = v.x; x[s][1] = v.y; x[s][2] = v.z; x[s][3] = v.w;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[s][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the largest component (Inf and NaN: none), kept where its inverse is a normal number too: a component in
        // [2^127, 2^128) becomes one in [2, 4)
        int e = (int)(__float_as_uint(top) >> 23) - 127;
        if (!(top > 0.f) || e > 127) e = 0;
        e = min(max(e, -126), 126);
        // The sums of codes (up to 2^15) meet the key's scale (up to 2^121, 2^125 in 4 bits) before the query's power of two.  Queries
        // so small that the product could leave the numbers though the score does not are held 9 places lower: their half
        // floats keep 2^-16 of the largest component (odd places of 4 bits: 2^-12), and numbers below 2^-126 whole.
        if (e < -20) e += 9;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
        float sum[GR];
#pragma unroll
        for (int i = 0; i < GR; ++i) sum[i] = 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            if constexpr (BITS == 8) {                    // one k-step per run
                qb[s][0] = pack_f16(x[s][0] * down, x[s][1] * down);
                qb[s][1] = pack_f16(x[s][2] * down, x[s][3] * down);
                const float2 a = unpack_f16(qb[s][0]), b = unpack_f16(qb[s][1]);
                sum[0] -= 1152.f * ((a.x + a.y) + (b.x + b.y));
            } else {                                      // k-steps (group, 0) and (group, 1) of runs 2t, 2t + 1
                const int gr = s >> 1, i = (s & 1) * 2;   // components i and i + 1 of both runs
                qb[s][0] = pack_f16(x[2 * gr][i] * down, x[2 * gr + 1][i] * down);
                qb[s][1] = pack_f16(x[2 * gr][i + 1] * down * 0.0625f, x[2 * gr + 1][i + 1] * down * 0.0625f);
                const float2 a = unpack_f16(qb[s][0]), b = unpack_f16(qb[s][1]);
                sum[gr] -= 1032.f * (a.x + a.y) + 1152.f * (b.x + b.y);
            }
        }
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
            off[i][0] = __shfl_sync(0xffffffffu, sum[i], 8 * t);          // head 2t: lanes 4 (2t) ..
            off[i][1] = __shfl_sync(0xffffffffu, sum[i], 8 * t + 4);
        }
        const float qs = up * scale_log2;
        qsA = __shfl_sync(0xffffffffu, qs, 8 * t);
        qsB = __shfl_sync(0xffffffffu, qs, 8 * t + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        mA = mB = NEG_BIG;
#pragma unroll
        for (int i = 0; i < GR; ++i) { rA[i] = rB[i] = NEG_BIG; fA[i] = fB[i] = 0.f; }
        lA = lB = 0.f;
    }

    // scores of keys g, g + 8 for heads 2t, 2t + 1: z = (A, g), (B, g), (A, g + 8), (B, g + 8), in base 2
    __device__ __forceinline__ void scores(const RawTile<BITS> &r, float (&z)[4]) const {
        if constexpr (BITS == 8) {
            float c[4] = {off[0][0], off[0][1], off[0][0], off[0][1]}, c2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const uint32_t w0 = word(r.k[0][s >> 2], s & 3), w1 = word(r.k[1][s >> 2], s & 3);
                mma_f16_16816(s & 1 ? c2 : c, __byte_perm(w0, F16_1024, 0x5150), __byte_perm(w1, F16_1024, 0x5150),
                              __byte_perm(w0, F16_1024, 0x5352), __byte_perm(w1, F16_1024, 0x5352), qb[s][0], qb[s][1]);
            }
            const float k0 = bf16_low(r.s[0]), k1 = bf16_low(r.s[1]);
            z[0] = (c[0] + c2[0]) * k0 * qsA; z[1] = (c[1] + c2[1]) * k0 * qsB;
            z[2] = (c[2] + c2[2]) * k1 * qsA; z[3] = (c[3] + c2[3]) * k1 * qsB;
        } else {
            z[0] = z[1] = z[2] = z[3] = 0.f;
#pragma unroll
            for (int gr = 0; gr < 4; ++gr) {
                const uint32_t sel = gr & 1 ? 0x7632 : 0x5410;
                uint32_t a = gr < 2 ? __byte_perm(r.k[0].x, r.k[0].z, sel) : __byte_perm(r.k[0].y, r.k[0].w, sel);
                uint32_t b = gr < 2 ? __byte_perm(r.k[1].x, r.k[1].z, sel) : __byte_perm(r.k[1].y, r.k[1].w, sel);
                float c[4];
                mma_f16_16816(c, and_or(a, 0x000f000fu, F16_1024), and_or(b, 0x000f000fu, F16_1024),
                              and_or(a, 0x00f000f0u, F16_1024), and_or(b, 0x00f000f0u, F16_1024), qb[2 * gr][0], qb[2 * gr][1],
                              {off[gr][0], off[gr][1], off[gr][0], off[gr][1]});
                a >>= 8; b >>= 8;
                mma_f16_16816(c, and_or(a, 0x000f000fu, F16_1024), and_or(b, 0x000f000fu, F16_1024),
                              and_or(a, 0x00f000f0u, F16_1024), and_or(b, 0x00f000f0u, F16_1024), qb[2 * gr + 1][0],
                              qb[2 * gr + 1][1]);
                const uint32_t s0 = gr < 2 ? r.s[0].x : r.s[0].y, s1 = gr < 2 ? r.s[1].x : r.s[1].y;
                const float k0 = gr & 1 ? bf16_high(s0) : bf16_low(s0), k1 = gr & 1 ? bf16_high(s1) : bf16_low(s1);
                z[0] = fmaf(c[0], k0, z[0]); z[1] = fmaf(c[1], k0, z[1]);
                z[2] = fmaf(c[2], k1, z[2]); z[3] = fmaf(c[3], k1, z[3]);
            }
            z[0] *= qsA; z[1] *= qsB; z[2] *= qsA; z[3] *= qsB;
        }
    }

    // value scale of a row's group
    static __device__ __forceinline__ float value_scale(const RawTile<BITS> &r, int row, int gr) {
        if constexpr (BITS == 8) return bf16_high(r.s[row]);
        else {
            const uint32_t w = gr < 2 ? r.s[row].z : r.s[row].w;
            return gr & 1 ? bf16_high(w) : bf16_low(w);
        }
    }

    // A fragment pair of one m-tile from the codes of two keys x, y: components (row g, row g + 8)
    __device__ __forceinline__ void pair8(uint32_t x, uint32_t y, bool high, uint32_t &a, uint32_t &b) const {
        const uint32_t p = __byte_perm(x, y, high ? 0x7362 : 0x5140);     // x_i, y_i, x_i+1, y_i+1
        a = hsub(__byte_perm(p, F16_1024, 0x5150), 1152.f);
        b = hsub(__byte_perm(p, F16_1024, 0x5352), 1152.f);
    }

    // Raise the accumulators' references to what these positions need; z: their scores, in base 2.
    template <int U>
    __device__ __forceinline__ void raise(const RawTile<BITS> (&r)[U], const float (&z)[U][4]) {
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
            float yA = NEG_BIG, yB = NEG_BIG;              // largest score + log2 of the value's scale
#pragma unroll
            for (int u = 0; u < U; ++u) {                  // (-inf for values of zero: they never raise r)
                const float v0 = log2_scale(fabsf(value_scale(r[u], 0, gr))), v1 = log2_scale(fabsf(value_scale(r[u], 1, gr)));
                yA = fmaxf(yA, fmaxf(z[u][0] + v0, z[u][2] + v1)); yB = fmaxf(yB, fmaxf(z[u][1] + v0, z[u][3] + v1));
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                yA = fmaxf(yA, __shfl_xor_sync(0xffffffffu, yA, o));
                yB = fmaxf(yB, __shfl_xor_sync(0xffffffffu, yB, o));
            }
            // (weights of 16 now; r no further below m than a float's exponent reaches with a weight of 2^8)
            const float sA = fmaxf(fmaxf(rA[gr], yA - 4.f), mA - 118.f), sB = fmaxf(fmaxf(rB[gr], yB - 4.f), mB - 118.f);
            const float alA = fast_exp2(rA[gr] - sA), alB = fast_exp2(rB[gr] - sB);
            rA[gr] = sA; rB[gr] = sB;
            fA[gr] = fast_exp2(mA - sA); fB[gr] = fast_exp2(mB - sB);
#pragma unroll
            for (int j = gr * (8 / GR); j < (gr + 1) * (8 / GR); ++j) {
                acc[j][0] *= alA; acc[j][1] *= alB;
                acc[j][2] *= alA; acc[j][3] *= alB;
            }
        }
    }

    // U blocks of 16 positions, `left` positions cached (16 U or more: all)
    template <int U>
    __device__ __forceinline__ void consume(const RawTile<BITS> (&r)[U], float (&z)[U][4], int left) {
        if (left < 16 * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (g + 16 * u >= left) z[u][0] = z[u][1] = NEG_BIG;
                if (g + 8 + 16 * u >= left) z[u][2] = z[u][3] = NEG_BIG;
            }
        }
        float tA = NEG_BIG, tB = NEG_BIG;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            tA = fmaxf(tA, fmaxf(z[u][0], z[u][2])); tB = fmaxf(tB, fmaxf(z[u][1], z[u][3]));
        }
        bool up = __any_sync(0xffffffffu, fmaxf(tA - mA, tB - mB) > 8.f);
        if (up) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                tA = fmaxf(tA, __shfl_xor_sync(0xffffffffu, tA, o)); tB = fmaxf(tB, __shfl_xor_sync(0xffffffffu, tB, o));
            }
            const float nA = fmaxf(mA, tA), nB = fmaxf(mB, tB);
            lA *= fast_exp2(mA - nA); lB *= fast_exp2(mB - nB);
            mA = nA; mB = nB;
        }
        float w[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u][0] = fast_exp2(z[u][0] - mA); w[u][1] = fast_exp2(z[u][1] - mB);
            w[u][2] = fast_exp2(z[u][2] - mA); w[u][3] = fast_exp2(z[u][3] - mB);
            if (left < 16 * U) {
                if (g + 16 * u >= left) w[u][0] = w[u][1] = 0.f;
                if (g + 8 + 16 * u >= left) w[u][2] = w[u][3] = 0.f;
            }
            lA += w[u][0] + w[u][2]; lB += w[u][1] + w[u][3];
        }
        // Weights times value scales as half floats; again with raised references where one of them is beyond 2^15.
        uint32_t pw[U][GR][2];
        auto weigh = [&]() {
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    const float2 f = make_float2(fA[gr], fB[gr]);
                    const float2 x = mul2(make_float2(w[u][0], w[u][1]), f), y = mul2(make_float2(w[u][2], w[u][3]), f);
                    const float s0 = value_scale(r[u], 0, gr), s1 = value_scale(r[u], 1, gr);
                    pw[u][gr][0] = pack_f16(x.x * s0, x.y * s0);
                    pw[u][gr][1] = pack_f16(y.x * s1, y.y * s1);
                    top = hmax(hmax(top, pw[u][gr][0]), pw[u][gr][1]);
                }
            return ((top + 0x07ff07ffu) & 0x80008000u) != 0;
        };
        if (__any_sync(0xffffffffu, weigh() || up)) {
            raise(r, z);
            weigh();
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) {
                const uint32_t b0 = movmatrix_trans(pw[u][gr][0]), b1 = movmatrix_trans(pw[u][gr][1]);
                if constexpr (BITS == 8) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t a0, a1, a2, a3;
                        pair8(word(r[u].v[0], j >> 1), word(r[u].v[1], j >> 1), j & 1, a0, a1);
                        pair8(word(r[u].v[2], j >> 1), word(r[u].v[3], j >> 1), j & 1, a2, a3);
                        mma_f16_16816(acc[j], a0, a1, a2, a3, b0, b1);
                    }
                } else {
                    const uint32_t sel = gr & 1 ? 0x7632 : 0x5410;
                    uint32_t x = gr < 2 ? __byte_perm(r[u].v[0].x, r[u].v[1].x, sel) : __byte_perm(r[u].v[0].y, r[u].v[1].y, sel);
                    uint32_t y = gr < 2 ? __byte_perm(r[u].v[2].x, r[u].v[3].x, sel) : __byte_perm(r[u].v[2].y, r[u].v[3].y, sel);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        mma_f16_16816(acc[2 * gr + i], hsub(and_or(x, 0x000f000fu, F16_1024), 1032.f),
                                      hfma(and_or(x, 0x00f000f0u, F16_1024), 0.0625f, -72.f),
                                      hsub(and_or(y, 0x000f000fu, F16_1024), 1032.f),
                                      hfma(and_or(y, 0x00f000f0u, F16_1024), 0.0625f, -72.f), b0, b1);
                        x >>= 8; y >>= 8;
                    }
                }
            }
    }

    // leave this warp's (sums, maximum, sum of weights) of heads < G in red[(warp * G + head) * 132 ..]
    __device__ __forceinline__ void store_partial(float *red, int warp, int G) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            lA += __shfl_xor_sync(0xffffffffu, lA, o);
            lB += __shfl_xor_sync(0xffffffffu, lB, o);
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int head = 2 * t + which;
            if (head >= G) continue;
            float *o = red + (warp * G + head) * 132;
            // back to weights relative to m, in two steps: values near the largest numbers have 2^(r - m) beyond them
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int d = BITS == 8 ? 16 * g + 2 * j : 32 * (j >> 1) + 4 * g + 2 * (j & 1), gr = j / (8 / GR);
                const float up = fast_exp2(0.5f * (which ? rB[gr] - mB : rA[gr] - mA));
                *reinterpret_cast<float2 *>(o + d) = make_float2(acc[j][which] * up * up, acc[j][2 + which] * up * up);
            }
            if (g == 0) { o[128] = which ? mB : mA; o[129] = which ? lB : lA; }
        }
    }
};

__device__ __forceinline__ void cp_async4(void *smem_dst, const void *gsrc, int src_bytes) {
    const unsigned dst = static_cast<unsigned>(__cvta_generic_to_shared(smem_dst));
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(gsrc), "r"(src_bytes));
}

// One warp's ring in shared memory: STAGES tiles of 16 U positions.  8 bits: the 16-byte chunk c of row r lies at place
// c ^ (r % 8) of the row's 128 bytes.  4 bits: two rows share 128 bytes, chunk c of row r lies at place
// (4 (r % 2) + c) ^ (2 (r / 2) % 8) of them.  Either way the eight lanes that read together meet no bank twice.
template <int BITS, int U, int STAGES>
struct Ring {
    using Q = Quant<BITS>;
    static constexpr int ROWS = 16 * U, CODES = ROWS * Q::ROW_BYTES, SCALES = ROWS * Q::SCALES * 2, BYTES = 2 * CODES + SCALES;
    unsigned char *base;
    int lane, copy;                                       // this lane's place in a tile as it is copied

    __device__ __forceinline__ explicit Ring(unsigned char *smem) : base(smem), lane(threadIdx.x & 31) {
        const int eight = lane >> 3;
        copy = eight * 128 + (((lane & 7) ^ (BITS == 8 ? eight : 2 * eight)) << 4);
    }
    // start the copies of a tile, `left` of its positions cached; k, v, s: where the tile begins in memory
    __device__ __forceinline__ void issue(int stage, const unsigned char *k, const unsigned char *v, const unsigned char *s,
                                          int left) {
        unsigned char *to = base + stage * BYTES;
        constexpr int PER = 512 / Q::ROW_BYTES;           // rows that the warp copies at once
        if (left >= ROWS) {                               // all but the last tile: nothing to ask about
#pragma unroll
            for (int i = 0; i < ROWS / PER; ++i) {
                const int at = i * 512 + (BITS == 8 ? copy ^ ((i & 1) << 6) : copy);
                cp_async16(to + at, k + i * 512 + lane * 16, 16);
                cp_async16(to + CODES + at, v + i * 512 + lane * 16, 16);
            }
            if (lane < ROWS) {
                if (BITS == 4) cp_async16(to + 2 * CODES + lane * 16, s + lane * 16, 16);
                else cp_async4(to + 2 * CODES + lane * 4, s + lane * 4, 4);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < ROWS / PER; ++i) {
            const bool ok = i * PER + lane / (32 / PER) < left;
            const int at = i * 512 + (BITS == 8 ? copy ^ ((i & 1) << 6) : copy);
            cp_async16(to + at, ok ? k + i * 512 + lane * 16 : k, ok ? 16 : 0);
            cp_async16(to + CODES + at, ok ? v + i * 512 + lane * 16 : v, ok ? 16 : 0);
        }
        if (lane < ROWS) {
            const bool ok = lane < left;
            if (BITS == 4) cp_async16(to + 2 * CODES + lane * 16, ok ? s + lane * 16 : s, ok ? 16 : 0);
            else cp_async4(to + 2 * CODES + lane * 4, ok ? s + lane * 4 : s, ok ? 4 : 0);
        }
    }
    __device__ __forceinline__ void keys(int stage, int u, RawTile<BITS> &r) const {
        const int g = lane >> 2, t = lane & 3;
        const unsigned char *k = base + stage * BYTES + u * 16 * Q::ROW_BYTES, *s = base + stage * BYTES + 2 * CODES;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (BITS == 8) {
                const unsigned char *row = k + (g + 8 * h) * 128;
                r.k[h][0] = *reinterpret_cast<const uint4 *>(row + ((2 * t ^ g) << 4));
                r.k[h][1] = *reinterpret_cast<const uint4 *>(row + (((2 * t + 1) ^ g) << 4));
                r.s[h] = *reinterpret_cast<const uint32_t *>(s + (16 * u + g + 8 * h) * 4);
            } else {
                r.k[h] = *reinterpret_cast<const uint4 *>(k + ((g >> 1) + 4 * h) * 128 + (((((g & 1) << 2) + t) ^ (g & 6)) << 4));
                r.s[h] = *reinterpret_cast<const uint4 *>(s + (16 * u + g + 8 * h) * 16);
            }
        }
    }
    __device__ __forceinline__ void values(int stage, int u, RawTile<BITS> &r) const {
        const int g = lane >> 2, t = lane & 3;
        const unsigned char *v = base + stage * BYTES + CODES + u * 16 * Q::ROW_BYTES;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                     // rows 2t, 2t + 1, 2t + 8, 2t + 9
            if constexpr (BITS == 8)
                r.v[i] = *reinterpret_cast<const uint4 *>(v + (2 * t + (i & 1) + 8 * (i >> 1)) * 128 +
                                                          ((g ^ (2 * t + (i & 1))) << 4));
            else
                r.v[i] = *reinterpret_cast<const uint2 *>(v + (t + 4 * (i >> 1)) * 128 +
                                                          (((((i & 1) << 2) + (g >> 1)) ^ (2 * t)) << 4) + (g & 1) * 8);
        }
    }
};

// Merge of heads with few partials, by warps: one warp a query head, all its partials asked for at once, a lane owns four
// columns.  (merge_head goes head by head, staging and synchronising: a CTA that had met two heads and merged both ended 7 us
// behind the others, 42.8 against 40.5 us for 16 ragged sequences of 8 heads with four query heads.)
constexpr int QUANT_FEW = 8;
template <typename Params>
__device__ __forceinline__ void merge_few(const Params &p, int row, int head, int parts, int64_t slot0) {
    const int lane = threadIdx.x & 31;
    const float *src = p.part + (slot0 * p.G + row) * PART_LD;
    float2 ml = make_float2(NEG_BIG, 0.f);
    if (lane < parts) ml = __ldcg(reinterpret_cast<const float2 *>(src + (int64_t)lane * p.G * PART_LD + HEAD_DIM));
    float4 a[QUANT_FEW];
#pragma unroll
    for (int i = 0; i < QUANT_FEW; ++i) {
        a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < parts) a[i] = __ldcg(reinterpret_cast<const float4 *>(src + (int64_t)i * p.G * PART_LD) + lane);
    }
    const float f = fast_exp2(ml.x - warp_max(ml.x));
    const float den = warp_sum(f * ml.y);
    float4 nm = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < QUANT_FEW; ++i) {
        if (i >= parts) break;
        const float fi = __shfl_sync(0xffffffffu, f, i);
        nm.x = fmaf(fi, a[i].x, nm.x); nm.y = fmaf(fi, a[i].y, nm.y);
        nm.z = fmaf(fi, a[i].z, nm.z); nm.w = fmaf(fi, a[i].w, nm.w);
    }
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + ((int64_t)head * p.G + row) * HEAD_DIM + lane * 4;
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack_bf16(quotient(p, nm.x, den), quotient(p, nm.y, den)),
                                                 pack_bf16(quotient(p, nm.z, den), quotient(p, nm.w, den)));
}

constexpr int QUANT_CTAS_PER_SM = 2;
constexpr int QUANT_MAX_SEG = 32;       // heads of a CTA whose partials wait in shared memory
// Rows of 132 floats of shared memory behind the rings: the warps' partials of one head of eight query heads, of two and
// more heads of fewer.  (The CTA that merges a head stages its partials over rings and rows alike.)
constexpr int QUANT_MOST_ROWS = 32;
static int quant_rows(int G) { return 8 * G < 16 ? 16 : 8 * G > QUANT_MOST_ROWS ? QUANT_MOST_ROWS : 8 * G; }

// The ways of sharing the work out, below, in blocks of 16 rows.  Measured on B200 (two query heads, 8-bit rows, us):
// ALONE: a head up to this long is left to one CTA, without a merge (400 rows: 7.8, in two parts 8.0; 1,000 rows: 10.2 and
//   8.8 in seven parts).  LEAST: blocks of a CTA at least, where a head is split (4: 9.1 for 1,000 rows).
// HOP: what the longest run of an even sharing may be beyond the average (64 heads of 256 blocks, 9 beyond it: even 17.7,
//   line 18.2; of 512 blocks, 17 beyond it: 30.6 and 28.2).
// START: what a head's start costs the CTA that meets it on the line (filling its rings anew, a second head to publish), as
//   if the head had so many blocks more (0 / 24 / 48: 40.5 / 39.8 / 39.4 for 16 ragged sequences of 8 heads, 70.8 / 68.7 /
//   70.0 for 64 heads of 2,048 blocks in 4 bits).
constexpr int QUANT_ALONE = 32, QUANT_LEAST = 8, QUANT_HOP = 16, QUANT_START = 24;

// (a * b - less) / c where the result fits 31 bits: a 32-bit quotient where the product allows it (all but billions of rows)
__device__ __forceinline__ int64_t mul_div(int64_t a, int64_t b, int64_t c, int less = 0) {
    const uint64_t ab = (uint64_t)a * (uint64_t)b - less;
    if ((ab >> 32) == 0 && (c >> 32) == 0) return (uint32_t)ab / (uint32_t)c;
    return (int64_t)(ab / (uint64_t)c);
}

// The rows of all heads, cut into blocks of 16, are shared out over the CTAs in one of two ways.
// Even: every head gets the same number of CTAs, each a run of its blocks.  It costs least where it leaves no CTA much more
//   than the average: no CTA serves two heads.
// Line: the blocks of all heads, each with QUANT_START empty places ahead of it, form one line and every CTA takes an equal
//   run of it, whatever the lengths; a run that meets only empty places of a head does not meet the head.  A head may be met
//   by several CTAs and a CTA may meet several heads; the partials of the pair (CTA c, head h) have slot c + h, which no two
//   pairs share (both only grow along the line), and a head's slots lie side by side.
// A CTA's warps take a quarter each of what the CTA has of a head and go on to the next head without waiting for one
// another; partials are combined, published and merged at the end (or when the shared memory for them is full).
// A head without rows counts one block, so that it gets its zeros.
struct QuantSegment {
    int head, split, parts;
    int64_t slot0;
};

template <int BITS, int U, int STAGES>
__global__ void __launch_bounds__(128, QUANT_CTAS_PER_SM) attend_quant_mma_kernel(const AttendQuantParams p) {
    using Q = Quant<BITS>;
    using Tiles = Ring<BITS, U, STAGES>;
    constexpr int WARPS = 4, ROWS = 16 * U, MAX_SEG = QUANT_MAX_SEG;
    extern __shared__ __align__(128) unsigned char smem[];    // the warps' rings, then rows x 132 floats
    float *const red = reinterpret_cast<float *>(smem + WARPS * STAGES * Tiles::BYTES);
    // (kept here, the tile loop needs the registers)
    __shared__ int64_t s_line, s_end, s_place[WARPS];     // where a warp's next head begins, and its first block there
    __shared__ int s_ctas, s_even, s_head[WARPS], s_b0[WARPS];
    __shared__ QuantSegment s_seg[MAX_SEG];
    __shared__ int s_last[MAX_SEG];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_trigger();
    const int group = p.n_group > 0 ? min(p.n_group, p.heads) : p.heads;
    const int groups = (p.heads + group - 1) / group;     // of heads that share one length
    auto blocks_of = [&](int i) {
        const int n = min(max(p.n_dev[i], 0), p.capacity);
        return max(1, (n + 15) >> 4);
    };
    auto heads_of = [&](int i) { return min(group, p.heads - i * group); };
    // Every warp for itself: blocks of the groups ahead of this lane's contiguous share of them, and the longest head
    const int share = (groups + 31) / 32;
    const int i0 = min(lane * share, groups), i1 = min(i0 + share, groups);
    int64_t mine = 0, before = 0, real;
    int longest = 0;
    if (groups == 1) {
        longest = blocks_of(0);
        real = (int64_t)longest * p.heads;
        if (lane == 0) mine = real;
    } else {
        for (int i = i0; i < i1; ++i) {
            const int b = blocks_of(i);
            mine += (int64_t)b * heads_of(i);
            longest = max(longest, b);
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        real = __shfl_sync(0xffffffffu, before, 31);
        before -= mine;
    }
    // CTAs per head, shared out evenly, and CTAs on the line
    const int each = longest <= QUANT_ALONE ? 1 : max(1, min(longest / QUANT_LEAST, (int)gridDim.x / p.heads));
    const int on_line = (int)max((int64_t)1, min((int64_t)gridDim.x, real / (2 * QUANT_LEAST)));
    const bool even = (int)gridDim.x >= p.heads && (longest + each - 1) / each <= mul_div(real, 1, on_line) + QUANT_HOP;
    const int ctas = even ? each * p.heads : on_line;
    if (blockIdx.x >= ctas) return;
    if (even) {
        const int head = blockIdx.x / each, part = blockIdx.x - head * each, b = blocks_of(head / group);
        const int parts = min(each, b);
        if (part >= parts) return;
        if (lane == 0) {
            s_head[warp] = head; s_place[warp] = 0;
            s_b0[warp] = (int)mul_div(b, part, parts);
            if (warp == 0) {
                s_end = mul_div(b, part + 1, parts);
                s_seg[0] = {head, part, parts, (int64_t)head * each};
            }
        }
    } else {
        const int64_t line = real + (int64_t)p.heads * QUANT_START, at = mul_div(line, blockIdx.x, ctas);
        before += (int64_t)i0 * group * QUANT_START;
        mine += i1 > i0 ? ((int64_t)(i1 - i0 - 1) * group + heads_of(i1 - 1)) * QUANT_START : 0;
        if (at >= before && at < before + mine) {         // exactly one lane
            int i = i0, b = blocks_of(i) + QUANT_START;
            int64_t one = (int64_t)b * heads_of(i);
            while (at >= before + one) { before += one; ++i; b = blocks_of(i) + QUANT_START; one = (int64_t)b * heads_of(i); }
            const int h = (int)mul_div(at - before, 1, b);
            const int64_t place = before + (int64_t)h * b;
            s_head[warp] = i * group + h; s_place[warp] = place; s_b0[warp] = (int)(at - place);
        }
        if (tid == 0) {
            s_line = line; s_ctas = ctas;
            s_end = mul_div(line, blockIdx.x + 1, ctas);
        }
    }
    if (tid == 0) s_even = even;
    __syncthreads();
    const int seg_cap = min(MAX_SEG, p.rows / (WARPS * p.G)), seg_floats = WARPS * p.G * PART_LD;
    Tiles ring(smem + warp * STAGES * Tiles::BYTES);
    for (bool more = true; more;) {
        int segs = 0;
        while (segs < seg_cap) {
            const int head = s_head[warp];
            const int64_t place = s_place[warp];
            more = place < s_end;
            if (!more) break;
            const int n = min(max(positions_of(p.n_dev, p.n_group, head), 0), p.capacity);
            const int start = s_even ? 0 : QUANT_START, blocks = max(1, (n + 15) >> 4);
            const int b0 = max(s_b0[warp] - start, 0), b1 = (int)min(s_end - place, (int64_t)(blocks + start)) - start;
            more = b1 > b0;
            if (!more) break;
            __syncwarp();
            if (lane == 0) {
                s_head[warp] = head + 1; s_place[warp] = place + blocks + start; s_b0[warp] = 0;
                if (warp == 0 && !s_even) {               // CTAs that meet this head: from its first block's to its last's
                    const int c0 = (int)mul_div(place + start + 1, s_ctas, s_line, 1);
                    const int c1 = (int)mul_div(place + start + blocks, s_ctas, s_line, 1);
                    s_seg[segs] = {head, (int)blockIdx.x - c0, c1 - c0 + 1, (int64_t)c0 + head};
                }
            }
            __syncwarp();
            // this warp's rows [r0, r1)
            const int per = (b1 - b0 + WARPS - 1) / WARPS;
            const int r0 = min((b0 + warp * per) * 16, n), r1 = min((b0 + min((warp + 1) * per, b1 - b0)) * 16, n);
            const int64_t row0 = (int64_t)head * p.capacity + r0;
            const unsigned char *k = p.kc + row0 * Q::ROW_BYTES, *v = p.vc + row0 * Q::ROW_BYTES;
            const unsigned char *s = reinterpret_cast<const unsigned char *>(p.scale) + row0 * Q::SCALES * 2;
            int ahead = r1 - r0, put = 0, get = 0;        // positions not asked for yet; stages
            auto more_rows = [&]() {
                if (ahead > 0) ring.issue(put, k, v, s, ahead);
                cp_async_commit();
                ahead -= ROWS;
                k += ROWS * Q::ROW_BYTES; v += ROWS * Q::ROW_BYTES; s += ROWS * Q::SCALES * 2;
                put = put + 1 == STAGES ? 0 : put + 1;
            };
#pragma unroll
            for (int i = 0; i < STAGES - 1; ++i) more_rows();
            WarpAttendQuant<BITS> wa;
            wa.init(static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)head * p.G * HEAD_DIM, p.G, p.scale_log2);
            for (int left = r1 - r0; left > 0; left -= ROWS) {
                more_rows();
                cp_async_wait<STAGES - 1>();
                __syncwarp();
                RawTile<BITS> r[U];
                float z[U][4];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    ring.keys(get, u, r[u]);
                    wa.scores(r[u], z[u]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) ring.values(get, u, r[u]);
                wa.consume(r, z, left);
                __syncwarp();                             // the stage may be filled again
                get = get + 1 == STAGES ? 0 : get + 1;
            }
            cp_async_wait<0>();
            wa.store_partial(red + segs * seg_floats, warp, p.G);
            ++segs;
        }
        __syncthreads();
        bool shared = false;
        for (int i = 0; i < segs; ++i) {
            publish_head<__nv_bfloat16>(p, red + i * seg_floats, WARPS, s_seg[i].head, s_seg[i].split, s_seg[i].parts,
                                        s_seg[i].slot0);
            shared |= s_seg[i].parts > 1;
        }
        if (shared) {
            __syncthreads();                              // the CTA's partials are on their way: one thread per head orders them
            if (tid < segs) {
                const int parts = s_seg[tid].parts;
                bool last = false;
                if (parts > 1) {
                    __threadfence();
                    last = atomicAdd(p.ticket + s_seg[tid].head, 1) == parts - 1;
                    __threadfence();
                    if (last) p.ticket[s_seg[tid].head] = 0;                   // ready for the next call on this stream
                }
                s_last[tid] = last;
            }
            __syncthreads();
            for (int i = 0; i < segs; ++i)
                if (s_last[i] && s_seg[i].parts > QUANT_FEW)
                    merge_head<__nv_bfloat16>(p, s_seg[i].head, s_seg[i].parts, s_seg[i].slot0, reinterpret_cast<float *>(smem),
                                              p.rows + WARPS * STAGES * Tiles::BYTES / (PART_LD * 4));
            for (int i = warp; i < segs * p.G; i += WARPS) {
                const QuantSegment &one = s_seg[i / p.G];
                if (s_last[i / p.G] && one.parts <= QUANT_FEW) merge_few(p, i % p.G, one.head, one.parts, one.slot0);
            }
        }
        __syncthreads();                                  // the next heads' partials go where these were
    }
}

template <int BITS, int U, int STAGES>
static int launch_quant_mma(const AttendQuantParams &p, cudaStream_t st) {
    auto kern = attend_quant_mma_kernel<BITS, U, STAGES>;
    constexpr int RINGS = 4 * STAGES * Ring<BITS, U, STAGES>::BYTES;
    constexpr int MOST = RINGS + QUANT_MOST_ROWS * PART_LD * 4;
    static_assert(QUANT_CTAS_PER_SM * (MOST + 4096) <= 227 * 1024, "the CTAs of an SM fit whatever the query heads");
    static bool configured[64] = {};       // the attribute is kept per device
    int dev = 0;
    SKV_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return SKV_E_RANGE;
    if (!configured[dev]) {
        SKV_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST));
        configured[dev] = true;
    }
    SKV_CUDA_OK(launch_early(kern, dim3(p.ctas), dim3(128), (size_t)RINGS + (size_t)p.rows * PART_LD * 4, st, p));
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

template <int BITS>
static int launch_quant_simple(const AttendQuantParams &p, cudaStream_t st) {
    const dim3 grid(p.splits, p.heads);
    if (p.G <= 1) attend_quant_simple_kernel<BITS, 1><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 2) attend_quant_simple_kernel<BITS, 2><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 4) attend_quant_simple_kernel<BITS, 4><<<grid, 128, 0, st>>>(p);
    else attend_quant_simple_kernel<BITS, 8><<<grid, 128, 0, st>>>(p);
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int skv_quant_ctas(void) { return QUANT_CTAS_PER_SM * device_sm_count(); }

extern "C" int64_t skv_quant_workspace_bytes(int heads, int G, int d, int ctas) {
    if (heads <= 0 || heads > 65535 || ctas <= 0 || ctas > 65535) return SKV_E_RANGE;
    if (d != HEAD_DIM || G < 1 || G > 8) return SKV_E_DIM;
    return ((int64_t)ctas + heads) * G * PART_LD * 4 + ((int64_t)heads * 4 + 255) / 256 * 256;
}

extern "C" int skv_attend_quant(const skv_qcache *c, const void *q, int dtype, int G, const int32_t *n_dev, int n_group,
                                void *out, void *workspace, int ctas, float scale, void *stream) {
    const int rc = qcache_check(c);
    if (rc) return rc;
    if (!q || !n_dev || !out || !workspace) return SKV_E_NULL;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    if (G < 1 || G > 8) return SKV_E_DIM;
    if (ctas <= 0 || ctas > 65535 || n_group < 0) return SKV_E_RANGE;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return SKV_E_ALIGN;
    AttendQuantParams p;
    p.heads = c->batch * c->h_kv; p.G = G; p.n_group = n_group; p.capacity = c->capacity;
    p.ctas = ctas; p.splits = (ctas + p.heads) / p.heads;
    p.rows = quant_rows(G);
    p.q = q; p.out = out; p.n_dev = n_dev;
    const QuantRows at = qcache_rows(c);
    p.kc = at.k; p.vc = at.v; p.scale = at.scale;
    p.part = static_cast<float *>(workspace);
    p.ticket = reinterpret_cast<int32_t *>(p.part + ((int64_t)ctas + p.heads) * G * PART_LD);
    p.scale_log2 = scale * LOG2E;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == SKV_F32) return c->bits == 8 ? launch_quant_simple<8>(p, st) : launch_quant_simple<4>(p, st);
    return c->bits == 8 ? launch_quant_mma<8, 2, 2>(p, st) : launch_quant_mma<4, 2, 3>(p, st);
}
