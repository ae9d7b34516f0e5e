// Attention of one new token per sequence over a prefix that all sequences share (its cache rows exist once) and over
// each sequence's own rows behind it.
//
// Simple kernel: a (sequence, KV head) pair walks the prefix and its own rows as one list, half a warp per row, float32
// arithmetic on the CUDA cores.
#include "skv_attend_finish.cuh"
#include "skv_common.cuh"

namespace skv {

struct PrefixParams {
    const void *q, *kp, *vp, *k, *v;
    const int32_t *n_dev;
    void *out;
    float *part;       // [batch * h_kv, splits, G, 132]
    int32_t *ticket;   // [batch * h_kv]
    int32_t *status;
    int batch, h_kv, G, n_group, prefix, rows_limit, splits;
    int64_t kph, kpr, vph, vpr, ksh, ksr, vsh, vsr;
    float scale_log2;
};

// Own rows of (sequence, KV head) `head`: its length, within the rows the cache has (a longer one is recorded).
__device__ __forceinline__ int own_rows(const PrefixParams &p, int head) {
    const int n = positions_of(p.n_dev, p.n_group, head);
    if (n > p.rows_limit && p.status && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status + head, SKV_ST_BAD_INDEX);
    return min(max(n, 0), p.rows_limit);
}

template <typename T, int GP>
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
        const bool shared = r < p.prefix;
        const int64_t own = r - p.prefix;
        const T *kr = shared ? static_cast<const T *>(p.kp) + h * p.kph + (int64_t)r * p.kpr
                             : static_cast<const T *>(p.k) + head * p.ksh + own * p.ksr;
        const T *vr = shared ? static_cast<const T *>(p.vp) + h * p.vph + (int64_t)r * p.vpr
                             : static_cast<const T *>(p.v) + head * p.vsh + own * p.vsr;
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
    finish_head<T>(p, red, 2 * WARPS, head, split, s_eff, (int64_t)head * p.splits, &s_flag, red, 2 * WARPS * GP);
}

template <typename T>
static int launch_prefix_simple(const PrefixParams &p, cudaStream_t st) {
    const dim3 grid(p.splits, p.batch * p.h_kv);
    if (p.G <= 1) attend_prefix_simple_kernel<T, 1><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 2) attend_prefix_simple_kernel<T, 2><<<grid, 128, 0, st>>>(p);
    else if (p.G <= 4) attend_prefix_simple_kernel<T, 4><<<grid, 128, 0, st>>>(p);
    else attend_prefix_simple_kernel<T, 8><<<grid, 128, 0, st>>>(p);
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int skv_prefix_splits(int batch, int h_kv, int G, int dtype) {
    if (batch <= 0 || h_kv <= 0 || (int64_t)batch * h_kv > 65535) return SKV_E_RANGE;
    if (G < 1 || G > 8) return SKV_E_DIM;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    return skv_attend_splits(batch * h_kv);
}

extern "C" int64_t skv_prefix_workspace_bytes(int batch, int h_kv, int G, int d, int splits) {
    if (batch <= 0 || h_kv <= 0) return SKV_E_RANGE;
    return skv_attend_workspace_bytes(batch * h_kv, G, d, splits);
}

extern "C" int skv_attend_prefix(const void *q, const void *k_prefix, const void *v_prefix, int prefix, const void *k,
                                 const void *v, const int32_t *n_dev, int n_group, void *out, void *workspace,
                                 int32_t *status, int batch, int h_kv, int G, int d, int dtype,
                                 int64_t kp_head_stride, int64_t kp_row_stride, int64_t vp_head_stride,
                                 int64_t vp_row_stride, int64_t k_head_stride, int64_t k_row_stride,
                                 int64_t v_head_stride, int64_t v_row_stride, int rows_limit, int splits, float scale,
                                 void *stream) {
    if (!q || !k || !v || !n_dev || !out || !workspace) return SKV_E_NULL;
    if (prefix > 0 && (!k_prefix || !v_prefix)) return SKV_E_NULL;
    if (d != HEAD_DIM) return SKV_E_DIM;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    if (G < 1 || G > 8) return SKV_E_DIM;
    if (batch <= 0 || h_kv <= 0 || (int64_t)batch * h_kv > 65535 || prefix < 0 || rows_limit < 0 ||
        (int64_t)prefix + rows_limit > 0x7fffffff - 64 || splits <= 0 || splits > 65535 || n_group < 0)
        return SKV_E_RANGE;
    const int per16 = dtype == SKV_BF16 ? 8 : 4;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(workspace) ||
        !aligned16(k_prefix) || !aligned16(v_prefix))
        return SKV_E_ALIGN;
    if (kp_head_stride % per16 || kp_row_stride % per16 || vp_head_stride % per16 || vp_row_stride % per16 ||
        k_head_stride % per16 || k_row_stride % per16 || v_head_stride % per16 || v_row_stride % per16 ||
        (prefix > 1 && (kp_row_stride < d || vp_row_stride < d)) || (rows_limit > 1 && (k_row_stride < d || v_row_stride < d)))
        return SKV_E_ALIGN;
    PrefixParams p;
    p.q = q; p.kp = k_prefix; p.vp = v_prefix; p.k = k; p.v = v; p.n_dev = n_dev; p.out = out; p.status = status;
    p.batch = batch; p.h_kv = h_kv; p.G = G; p.n_group = n_group; p.prefix = prefix; p.rows_limit = rows_limit;
    p.splits = splits;
    p.part = static_cast<float *>(workspace);
    p.ticket = reinterpret_cast<int32_t *>(p.part + (int64_t)batch * h_kv * splits * G * PART_LD);
    p.kph = kp_head_stride; p.kpr = kp_row_stride; p.vph = vp_head_stride; p.vpr = vp_row_stride;
    p.ksh = k_head_stride; p.ksr = k_row_stride; p.vsh = v_head_stride; p.vsr = v_row_stride;
    p.scale_log2 = scale * LOG2E;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == SKV_F32 ? launch_prefix_simple<float>(p, st) : launch_prefix_simple<__nv_bfloat16>(p, st);
}
