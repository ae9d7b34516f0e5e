// The end of a split attention: the warps' partials of a CTA are combined, published, and the last CTA of a head
// merges the head's partials into the output.  Shared by every attention kernel whose grid is (splits, heads).
#pragma once

#include "skv_attend_core.cuh"

namespace skv {

constexpr int PART_LD = 132;               // floats per partial row: 128 sums, max, sum, 2 unused

// Phase time stamp of a kernel's parameters: nothing unless the kernel overloads it for its own parameter type.
template <typename Params>
__device__ __forceinline__ void stamp(const Params &, int) {}

// A row's output: zero where no key had a weight.  A sum of weights that is no number counts as none, unless the kernel overloads
// it for its own parameter type.
template <typename Params>
__device__ __forceinline__ float quotient(const Params &, float num, float den) { return den > 0.f ? num / den : 0.f; }

// `p` needs: out, part [slots, G, 132], ticket [heads], G.  The head's s_eff partials lie in the slots from slot0 on; this
// CTA's is number `split` of them.
// blockDim.x is 128: one thread per output column.

// Combine the partial (max, sum, acc) sets that the warps of this CTA left in shared memory (red[set][g][132]: 128 acc,
// then max, sum): into the output where this CTA alone served the head, else into the CTA's slot.
template <typename T, typename Params>
__device__ __forceinline__ void publish_head(const Params &p, const float *red, int sets, int head, int split, int s_eff,
                                             int64_t slot0) {
    const int G = p.G, tid = threadIdx.x;
    T *out = static_cast<T *>(p.out);
    float *pa = p.part + (slot0 + split) * G * PART_LD;
#pragma unroll 1
    for (int g = 0; g < G; ++g) {
        float M = NEG_BIG;
        for (int w = 0; w < sets; ++w) M = fmaxf(M, red[(w * G + g) * 132 + 128]);
        float dn = 0.f, nm = 0.f;
        for (int w = 0; w < sets; ++w) {
            const float *r = red + (w * G + g) * 132;
            float f = fast_exp2(r[128] - M);
            dn += f * r[129];
            nm += f * r[tid];
        }
        if (s_eff == 1) {
            store_out(out + ((int64_t)head * G + g) * HEAD_DIM + tid, quotient(p, nm, dn));
        } else {
            __stcg(pa + g * PART_LD + tid, nm);
            if (tid == 0) __stcg(reinterpret_cast<float2 *>(pa + g * PART_LD + HEAD_DIM), make_float2(M, dn));
        }
    }
}

// Merge of the head's partials by the CTA that published last.  The partial rows are copied into the shared memory
// the CTA no longer needs with asynchronous 16-byte copies, all requested before any is used: one round
// trip to L2 where they fit (stage_rows rows), chunks of one query head's splits with a running maximum
// otherwise.  Up to four query heads are then folded at once, each by 4 / (their number) warps that share
// its rows; a lane owns four columns.
template <typename T, typename Params>
__device__ __forceinline__ void merge_head(const Params &p, int head, int s_eff, int64_t slot0, float *stg, int stage_rows) {
    const int G = p.G, tid = threadIdx.x;
    T *out = static_cast<T *>(p.out);
    __shared__ __align__(16) float s_sum[4][PART_LD];
    const int lane = tid & 31, wid = tid >> 5;
    const float *src = p.part + slot0 * G * PART_LD;
    const int gc = max(1, min(G, stage_rows / s_eff));        // query heads staged together
    const int cs = gc > 1 ? s_eff : min(s_eff, stage_rows);   // splits per chunk
    for (int g0 = 0; g0 < G; g0 += gc) {
        const int ng = min(gc, G - g0);
        float M = NEG_BIG, dn = 0.f;                           // carried over chunks only when ng == 1
        float4 nm = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < s_eff; s0 += cs) {
            const int ns = min(cs, s_eff - s0);
            if (ng == G) {                                     // every row of the head: one contiguous block
                const int chunks = ns * G * (PART_LD / 4);
                const float *blk = src + (int64_t)s0 * G * PART_LD;
                for (int c = tid; c < chunks; c += 128) cp_async16(stg + c * 4, blk + c * 4, 16);
            } else {                                           // rows of query heads [g0, g0 + ng) only
                for (int gi = 0; gi < ng; ++gi)
                    for (int i = wid; i < ns; i += 4) {
                        const float *row = src + ((int64_t)(s0 + i) * G + g0 + gi) * PART_LD;
                        float *dst = stg + (i * ng + gi) * PART_LD;
                        cp_async16(dst + lane * 4, row + lane * 4, 16);
                        if (lane == 0) cp_async16(dst + HEAD_DIM, row + HEAD_DIM, 16);
                    }
            }
            cp_async_commit();
            cp_async_wait<0>();
            __syncthreads();
            stamp(p, 7);
            // staged row of (split i, query head gi): stg + (i * ng + gi) * PART_LD
            const bool last_chunk = s0 + cs >= s_eff;
            for (int gb = 0; gb < ng; gb += 4) {
                const int nq = min(4, ng - gb), wpg = 4 / nq;
                const int gi = gb + wid / wpg, sub = wid % wpg;
                if (wid < nq * wpg) {
                    if (ng > 1) { M = NEG_BIG; dn = 0.f; nm = make_float4(0.f, 0.f, 0.f, 0.f); }
                    const float *rows = stg + gi * PART_LD;
                    const int ld = ng * PART_LD;
                    float mb = NEG_BIG;
                    for (int i = lane; i < ns; i += 32) mb = fmaxf(mb, rows[i * ld + HEAD_DIM]);
                    mb = fmaxf(M, warp_max(mb));
                    const float al = fast_exp2(M - mb);
                    M = mb;
                    dn *= al; nm.x *= al; nm.y *= al; nm.z *= al; nm.w *= al;
#pragma unroll 4
                    for (int i = sub; i < ns; i += wpg) {
                        const float2 ml = *reinterpret_cast<const float2 *>(rows + i * ld + HEAD_DIM);
                        const float4 a = *reinterpret_cast<const float4 *>(rows + i * ld + lane * 4);
                        const float f = fast_exp2(ml.x - M);
                        dn = fmaf(f, ml.y, dn);
                        nm.x = fmaf(f, a.x, nm.x); nm.y = fmaf(f, a.y, nm.y);
                        nm.z = fmaf(f, a.z, nm.z); nm.w = fmaf(f, a.w, nm.w);
                    }
                    *reinterpret_cast<float4 *>(&s_sum[wid][lane * 4]) = nm;
                    if (lane == 0) s_sum[wid][HEAD_DIM] = dn;
                }
                __syncthreads();
                if (ng > 1 || last_chunk)
                    for (int qi = 0; qi < nq; ++qi) {
                        float num = 0.f, den = 0.f;
                        for (int w = 0; w < wpg; ++w) {
                            num += s_sum[qi * wpg + w][tid];
                            den += s_sum[qi * wpg + w][HEAD_DIM];
                        }
                        store_out(out + ((int64_t)head * G + g0 + gb + qi) * HEAD_DIM + tid, quotient(p, num, den));
                    }
                __syncthreads();
            }
        }
    }
    if (tid == 0) p.ticket[head] = 0;     // ready for the next call on this stream
}

// Both, with the ticket between them: the last CTA of the head to publish merges.
template <typename T, typename Params>
__device__ __forceinline__ void finish_head(const Params &p, const float *red, int sets, int head, int split,
                                            int s_eff, int64_t slot0, int *sh_flag, float *stage,
                                            int stage_rows) {
    publish_head<T>(p, red, sets, head, split, s_eff, slot0);
    if (s_eff == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int t = atomicAdd(p.ticket + head, 1);
        *sh_flag = (t == s_eff - 1);
    }
    __syncthreads();
    stamp(p, 5);
    if (!*sh_flag) return;
    __threadfence();
    merge_head<T>(p, head, s_eff, slot0, stage, stage_rows);
    stamp(p, 6);
}

}  // namespace skv
