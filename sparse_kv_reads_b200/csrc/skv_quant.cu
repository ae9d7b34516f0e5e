// Writing rows into a quantised KV cache and reading them back.
//
// Both move a few bytes per value and compute little: HBM-bound for a prefill chunk, launch-bound for a decode step.
// Half a warp serves one cached position of one KV head, key and value together, so that a lane's two 16-byte loads (8
// values each) are requested before either is used and the position's scales are written by one place.
#include "skv_quant.cuh"
#include "skv_rope.cuh"

namespace skv {

struct RowsParams {
    void *k, *v;                 // source of a write, destination of a read (element strides below)
    int64_t kb, kh, kr, vb, vh, vr;
    unsigned char *kc, *vc;
    __nv_bfloat16 *scale;
    int32_t *status;
    const int64_t *pos;          // first position: pos[0], or pos[sequence] with pos_per_seq; null: pos0
    int64_t pos0;
    int pos_per_seq, batch, h_kv, capacity, tokens;
};

// Position of token `t` of sequence `b`; -1 (recorded in the head's status) when it lies outside the cache.
__device__ __forceinline__ int64_t row_position(const RowsParams &p, int b, int head, int t) {
    const int64_t first = p.pos ? p.pos[p.pos_per_seq ? b : 0] : p.pos0;
    const int64_t at = first + t;
    if (first < 0 || first > p.capacity || at >= p.capacity) {
        if (p.status) atomicOr(p.status + head, SKV_ST_BAD_INDEX);
        return -1;
    }
    return at;
}

template <typename T, int BITS>
__global__ void __launch_bounds__(256) quant_write_kernel(const RowsParams p) {
    using Q = Quant<BITS>;
    const int sub = threadIdx.x & 15;
    const unsigned hmask = (threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu;
    const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= (int64_t)p.batch * p.h_kv * p.tokens) return;         // uniform within the half warp
    const int t = (int)(item % p.tokens), head = (int)(item / p.tokens);
    const int b = head / p.h_kv, h = head % p.h_kv;
    const int64_t at = row_position(p, b, head, t);
    if (at < 0) return;
    float k[8], v[8];
    load8(static_cast<const T *>(p.k) + b * p.kb + h * p.kh + t * p.kr + sub * 8, k);
    load8(static_cast<const T *>(p.v) + b * p.vb + h * p.vh + t * p.vr + sub * 8, v);
    const int64_t row = (int64_t)head * p.capacity + at;
    const float ks = quantise_row8<BITS>(k, sub, hmask, p.kc + row * Q::ROW_BYTES, true);
    const float vs = quantise_row8<BITS>(v, sub, hmask, p.vc + row * Q::ROW_BYTES, true);
    if (sub % (16 / Q::GROUPS) == 0) {
        __nv_bfloat16 *s = p.scale + row * Q::SCALES + group_of<BITS>(sub);
        s[0] = __float2bfloat16(ks);
        s[Q::GROUPS] = __float2bfloat16(vs);
    }
}

__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
    __align__(16) __nv_bfloat162 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(o);
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// code * scale has at most 15 significant bits: exact in float32, rounded once where the destination is bf16.
template <typename T, int BITS>
__global__ void __launch_bounds__(256) quant_read_kernel(const RowsParams p) {
    using Q = Quant<BITS>;
    const int sub = threadIdx.x & 15;
    const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (item >= (int64_t)p.batch * p.h_kv * p.tokens) return;
    const int t = (int)(item % p.tokens), head = (int)(item / p.tokens);
    const int b = head / p.h_kv, h = head % p.h_kv;
    const int64_t at = row_position(p, b, head, t);
    float k[8] = {}, v[8] = {};
    if (at >= 0) {
        const int64_t row = (int64_t)head * p.capacity + at;
        const __nv_bfloat16 *s = p.scale + row * Q::SCALES + group_of<BITS>(sub);
        restore_row8<BITS>(p.kc + row * Q::ROW_BYTES, sub, __bfloat162float(s[0]), k);
        restore_row8<BITS>(p.vc + row * Q::ROW_BYTES, sub, __bfloat162float(s[Q::GROUPS]), v);
    }
    store8(static_cast<T *>(p.k) + b * p.kb + h * p.kh + t * p.kr + sub * 8, k);
    store8(static_cast<T *>(p.v) + b * p.vb + h * p.vh + t * p.vr + sub * 8, v);
}

// The decode step's QK-norm + rotary (qk_rope_cache_kernel's arithmetic and roundings) with the new key and value rows
// quantised into the cache.  One warp per (sequence, head): lane l owns components 4l .. 4l+3, one run of a 4-bit row.
template <int BITS>
__global__ void __launch_bounds__(128) qk_rope_quant_kernel(const __nv_bfloat16 *qkv, const __nv_bfloat16 *qw,
                                                            const __nv_bfloat16 *kw, const __nv_bfloat16 *cos_t,
                                                            const __nv_bfloat16 *sin_t, __nv_bfloat16 *q_out, int H,
                                                            float eps, const RowsParams p) {
    using Q = Quant<BITS>;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5);
    const int per = H + 2 * p.h_kv;
    if (item >= p.batch * per) return;
    const int b = item / per, j = item % per;
    const int head = b * p.h_kv + (j < H ? j / (H / p.h_kv) : (j - H) % p.h_kv);
    const int64_t pos = row_position(p, b, head, 0);
    if (pos < 0) return;                                              // recorded; the tables have `capacity` rows at least
    const __nv_bfloat16 *src = qkv + ((int64_t)b * per + j) * HEAD_DIM;
    float4 r;
    if (j >= H + p.h_kv) r = load4(src + lane * 4);
    else r = norm_rope_head(src, j < H ? qw : kw, cos_t + pos * HEAD_DIM, sin_t + pos * HEAD_DIM, eps, lane);
    if (j < H) {
        store_bf16x4(q_out + ((int64_t)b * H + j) * HEAD_DIM + lane * 4, r);
        return;
    }
    const bool is_v = j >= H + p.h_kv;
    const int64_t row = (int64_t)head * p.capacity + pos;
    uint32_t top = max(max(magnitude_bits(r.x), magnitude_bits(r.y)), max(magnitude_bits(r.z), magnitude_bits(r.w)));
#pragma unroll
    for (int o = 1; o < (BITS == 8 ? 32 : 8); o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s = group_scale<BITS>(top);
    const uint32_t c0 = stored_code<BITS>(r.x, s), c1 = stored_code<BITS>(r.y, s), c2 = stored_code<BITS>(r.z, s),
                   c3 = stored_code<BITS>(r.w, s);
    unsigned char *dst = (is_v ? p.vc : p.kc) + row * Q::ROW_BYTES;
    if (BITS == 8) *reinterpret_cast<uint32_t *>(dst + lane * 4) = c0 | c1 << 8 | c2 << 16 | c3 << 24;
    else *reinterpret_cast<uint16_t *>(dst + ((lane & 7) * 4 + (lane >> 3)) * 2) = (uint16_t)(c0 | c1 << 4 | c2 << 8 | c3 << 12);
    if (lane % (32 / Q::GROUPS) == 0)
        p.scale[row * Q::SCALES + (is_v ? Q::GROUPS : 0) + lane / (32 / Q::GROUPS)] = __float2bfloat16(s);
}

static int rows_check(const skv_qcache *c, const void *k, const void *v, int dtype, int batch, int tokens, int64_t kb,
                      int64_t kh, int64_t kr, int64_t vb, int64_t vh, int64_t vr, const int64_t *pos, int64_t pos0,
                      RowsParams &p) {
    const int rc = qcache_check(c);
    if (rc) return rc;
    if (!k || !v) return SKV_E_NULL;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    if (batch <= 0 || batch > c->batch || tokens < 0 || tokens > c->capacity) return SKV_E_RANGE;
    if (!pos && (pos0 < 0 || pos0 + tokens > c->capacity)) return SKV_E_RANGE;
    const int per16 = dtype == SKV_BF16 ? 8 : 4;
    if (!aligned16(k) || !aligned16(v) || kb % per16 || kh % per16 || kr % per16 || vb % per16 || vh % per16 || vr % per16)
        return SKV_E_ALIGN;
    p.k = const_cast<void *>(k); p.v = const_cast<void *>(v);
    p.kb = kb; p.kh = kh; p.kr = kr; p.vb = vb; p.vh = vh; p.vr = vr;
    p.kc = static_cast<unsigned char *>(c->k); p.vc = static_cast<unsigned char *>(c->v);
    p.scale = static_cast<__nv_bfloat16 *>(c->scale); p.status = c->status;
    p.pos = pos; p.pos0 = pos0;
    p.batch = batch; p.h_kv = c->h_kv; p.capacity = c->capacity; p.tokens = tokens;
    return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int skv_quant_write(const skv_qcache *c, const void *k, const void *v, int dtype, int batch, int tokens,
                               int64_t k_batch_stride, int64_t k_head_stride, int64_t k_row_stride,
                               int64_t v_batch_stride, int64_t v_head_stride, int64_t v_row_stride, const int64_t *pos,
                               int pos_per_seq, int64_t pos0, void *stream) {
    RowsParams p;
    const int rc = rows_check(c, k, v, dtype, batch, tokens, k_batch_stride, k_head_stride, k_row_stride, v_batch_stride,
                              v_head_stride, v_row_stride, pos, pos0, p);
    if (rc) return rc;
    if (tokens == 0) return SKV_OK;
    p.pos_per_seq = pos_per_seq;
    const int64_t items = (int64_t)batch * c->h_kv * tokens;
    const dim3 grid((unsigned)((items + 15) / 16));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == SKV_BF16 && c->bits == 8) quant_write_kernel<__nv_bfloat16, 8><<<grid, 256, 0, st>>>(p);
    else if (dtype == SKV_BF16) quant_write_kernel<__nv_bfloat16, 4><<<grid, 256, 0, st>>>(p);
    else if (c->bits == 8) quant_write_kernel<float, 8><<<grid, 256, 0, st>>>(p);
    else quant_write_kernel<float, 4><<<grid, 256, 0, st>>>(p);
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

extern "C" int skv_quant_read(const skv_qcache *c, void *k, void *v, int dtype, int batch, int tokens,
                              int64_t k_batch_stride, int64_t k_head_stride, int64_t k_row_stride,
                              int64_t v_batch_stride, int64_t v_head_stride, int64_t v_row_stride, const int64_t *pos,
                              int pos_per_seq, int64_t pos0, void *stream) {
    RowsParams p;
    const int rc = rows_check(c, k, v, dtype, batch, tokens, k_batch_stride, k_head_stride, k_row_stride, v_batch_stride,
                              v_head_stride, v_row_stride, pos, pos0, p);
    if (rc) return rc;
    if (tokens == 0) return SKV_OK;
    p.pos_per_seq = pos_per_seq;
    const int64_t items = (int64_t)batch * c->h_kv * tokens;
    const dim3 grid((unsigned)((items + 15) / 16));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == SKV_BF16 && c->bits == 8) quant_read_kernel<__nv_bfloat16, 8><<<grid, 256, 0, st>>>(p);
    else if (dtype == SKV_BF16) quant_read_kernel<__nv_bfloat16, 4><<<grid, 256, 0, st>>>(p);
    else if (c->bits == 8) quant_read_kernel<float, 8><<<grid, 256, 0, st>>>(p);
    else quant_read_kernel<float, 4><<<grid, 256, 0, st>>>(p);
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

extern "C" int skv_qk_rope_quant(const skv_qcache *c, const void *qkv, const void *q_norm_w, const void *k_norm_w,
                                 const void *cos_table, const void *sin_table, const int64_t *pos, int pos_per_seq,
                                 void *q_out, int batch, int H, float eps, void *stream) {
    RowsParams p = {};
    if (!qkv || !q_norm_w || !k_norm_w || !cos_table || !sin_table || !pos || !q_out) return SKV_E_NULL;
    const int rc = rows_check(c, qkv, qkv, SKV_BF16, batch, 1, 0, 0, 0, 0, 0, 0, pos, 0, p);
    if (rc) return rc;
    if (H <= 0 || H % c->h_kv) return SKV_E_RANGE;
    if (!aligned16(q_norm_w) || !aligned16(k_norm_w) || !aligned16(q_out) || !aligned16(cos_table) || !aligned16(sin_table))
        return SKV_E_ALIGN;
    p.pos_per_seq = pos_per_seq;
    const int items = batch * (H + 2 * c->h_kv);
    auto kern = c->bits == 8 ? qk_rope_quant_kernel<8> : qk_rope_quant_kernel<4>;
    SKV_CUDA_OK(launch_pdl(kern, dim3((items + 3) / 4), dim3(128), 0, static_cast<cudaStream_t>(stream),
                           static_cast<const __nv_bfloat16 *>(qkv), static_cast<const __nv_bfloat16 *>(q_norm_w),
                           static_cast<const __nv_bfloat16 *>(k_norm_w), static_cast<const __nv_bfloat16 *>(cos_table),
                           static_cast<const __nv_bfloat16 *>(sin_table), static_cast<__nv_bfloat16 *>(q_out), H, eps, p));
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}
