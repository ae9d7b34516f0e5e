// Attention of one new token per sequence over a quantised KV cache, split over CTAs, merged by the last CTA of a head.
//
// Simple kernel: half a warp per row, float32 arithmetic on the CUDA cores.
#include "skv_attend_finish.cuh"
#include "skv_quant.cuh"

namespace skv {

struct AttendQuantParams {
    const void *q;
    const unsigned char *kc, *vc;
    const __nv_bfloat16 *scale;
    const int32_t *n_dev;
    void *out;
    float *part;       // [heads, splits, G, 132]
    int32_t *ticket;   // [heads]
    int heads, G, n_group, capacity, splits;
    float scale_log2;
};

template <typename T, int BITS, int GP>
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
    const T *q = static_cast<const T *>(p.q) + (int64_t)head * G * HEAD_DIM;

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
    finish_head<T>(p, red, 2 * WARPS, head, split, s_eff, &s_flag, red, 2 * WARPS * GP);
}

template <typename T, int BITS>
static int launch_quant_simple(const AttendQuantParams &p, cudaStream_t st) {
    const dim3 grid(p.splits, p.heads);
    if (p.G <= 1) attend_quant_simple_kernel<T, BITS, 1><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 2) attend_quant_simple_kernel<T, BITS, 2><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 4) attend_quant_simple_kernel<T, BITS, 4><<<grid, 128, 0, st>>>(p);
    else attend_quant_simple_kernel<T, BITS, 8><<<grid, 128, 0, st>>>(p);
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int skv_attend_quant(const skv_qcache *c, const void *q, int dtype, int G, const int32_t *n_dev, int n_group,
                                void *out, void *workspace, int splits, float scale, void *stream) {
    const int rc = qcache_check(c);
    if (rc) return rc;
    if (!q || !n_dev || !out || !workspace) return SKV_E_NULL;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    if (G < 1 || G > 8) return SKV_E_DIM;
    if (splits <= 0 || splits > 65535 || n_group < 0) return SKV_E_RANGE;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return SKV_E_ALIGN;
    AttendQuantParams p;
    p.heads = c->batch * c->h_kv; p.G = G; p.n_group = n_group; p.capacity = c->capacity; p.splits = splits;
    p.q = q; p.out = out; p.n_dev = n_dev;
    p.kc = static_cast<const unsigned char *>(c->k); p.vc = static_cast<const unsigned char *>(c->v);
    p.scale = static_cast<const __nv_bfloat16 *>(c->scale);
    p.part = static_cast<float *>(workspace);
    p.ticket = reinterpret_cast<int32_t *>(p.part + (int64_t)p.heads * splits * G * PART_LD);
    p.scale_log2 = scale * LOG2E;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == SKV_F32) return c->bits == 8 ? launch_quant_simple<float, 8>(p, st) : launch_quant_simple<float, 4>(p, st);
    return c->bits == 8 ? launch_quant_simple<__nv_bfloat16, 8>(p, st) : launch_quant_simple<__nv_bfloat16, 4>(p, st);
}
