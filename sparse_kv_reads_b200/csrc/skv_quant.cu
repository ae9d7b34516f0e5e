// Writing rows into a quantised KV cache and reading them back.
//
// Both move a few bytes per value and compute little: HBM-bound for a prefill chunk, launch-bound for a decode step.
// Half a warp serves one cached position of one KV head, key and value together (a lane has 8 values of each), and two
// positions at once, so that a lane's four loads are requested before any is used.
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
    uint32_t items;              // positions x heads x sequences
    int flat;                    // the grid is flat over them, else (positions, KV heads, sequences)
};

constexpr int AT_ONCE = 2;       // positions of a half warp
constexpr int PER_CTA = 16 * AT_ONCE;

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

// Where the work of a half warp lies: 3-d grid (positions, KV heads, sequences), or, for few tokens per sequence, a flat one.
struct Place {
    int b, h, t, head;
    bool any;
};
__device__ __forceinline__ Place place_of(const RowsParams &p, int r) {
    Place w;
    const uint32_t item = blockIdx.x * PER_CTA + r * 16 + (threadIdx.x >> 4);
    if (p.flat) {
        const uint32_t head = item / (uint32_t)p.tokens;
        w.any = item < p.items;
        w.t = (int)(item - head * p.tokens);
        w.head = (int)head;
        w.b = (int)(head / (uint32_t)p.h_kv);
        w.h = w.head - w.b * p.h_kv;
    } else {
        w.any = item < (uint32_t)p.tokens;
        w.t = (int)item;
        w.h = blockIdx.y;
        w.b = blockIdx.z;
        w.head = w.b * p.h_kv + w.h;
    }
    return w;
}

// A lane's eight values of a key or value row.
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { v = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void values(float (&x)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    // the largest magnitude in both halves' order of the packed numbers (NaN above all)
    __device__ __forceinline__ __nv_bfloat162 largest() const {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
        return __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = __ldcs(reinterpret_cast<const float4 *>(p));
        b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};

// The scales of the lane's groups of key and value: over 16 lanes (8 bits) or 4 (4 bits).
template <int BITS>
__device__ __forceinline__ void scales_of(const Eight<__nv_bfloat16> &k, const Eight<__nv_bfloat16> &v, unsigned hmask, float &ks,
                                          float &vs) {
    const __nv_bfloat162 tk = k.largest(), tv = v.largest();
    __nv_bfloat162 top = __hmax2_nan(__lows2bfloat162(tk, tv), __highs2bfloat162(tk, tv));      // (key, value)
#pragma unroll
    for (int o = 1; o < (BITS == 8 ? 16 : 4); o <<= 1) {
        const uint32_t u = __shfl_xor_sync(hmask, *reinterpret_cast<const uint32_t *>(&top), o, 16);
        top = __hmax2_nan(top, *reinterpret_cast<const __nv_bfloat162 *>(&u));
    }
    const uint32_t u = *reinterpret_cast<const uint32_t *>(&top);
    ks = group_scale_bf16<BITS>(u << 16 & 0x7fffffffu);
    vs = group_scale_bf16<BITS>(u & 0x7fff0000u);
}
template <int BITS>
__device__ __forceinline__ void scales_of(const Eight<float> &k, const Eight<float> &v, unsigned hmask, float &ks, float &vs) {
    float x[8], y[8];
    k.values(x);
    v.values(y);
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { a = max(a, magnitude_bits(x[i])); b = max(b, magnitude_bits(y[i])); }
#pragma unroll
    for (int o = 1; o < (BITS == 8 ? 16 : 4); o <<= 1) {
        a = max(a, __shfl_xor_sync(hmask, a, o, 16));
        b = max(b, __shfl_xor_sync(hmask, b, o, 16));
    }
    ks = group_scale<BITS>(a);
    vs = group_scale<BITS>(b);
}

template <typename T, int BITS>
__global__ void __launch_bounds__(256) quant_write_kernel(const RowsParams p) {
    using Q = Quant<BITS>;
    constexpr bool EXACT = sizeof(T) == 4;
    const int sub = threadIdx.x & 15;
    const unsigned hmask = (threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu;
    Eight<T> k[AT_ONCE], v[AT_ONCE];
    int64_t row[AT_ONCE];
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {                    // (everything about a position is uniform within its half warp)
        const Place w = place_of(p, r);
        row[r] = -1;
        if (!w.any) continue;
        const int64_t at = row_position(p, w.b, w.head, w.t);
        if (at < 0) continue;
        row[r] = (int64_t)w.head * p.capacity + at;
        k[r].load(static_cast<const T *>(p.k) + w.b * p.kb + w.h * p.kh + w.t * p.kr + sub * 8);
        v[r].load(static_cast<const T *>(p.v) + w.b * p.vb + w.h * p.vh + w.t * p.vr + sub * 8);
    }
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {
        if (row[r] < 0) continue;
        float ks, vs, x[8];
        uint32_t c[8];
        scales_of<BITS>(k[r], v[r], hmask, ks, vs);
        k[r].values(x);
        stored_codes<BITS, EXACT>(x, ks, c);
        const uint2 kc = packed_codes<BITS>(c);
        v[r].values(x);
        stored_codes<BITS, EXACT>(x, vs, c);
        const uint2 vc = packed_codes<BITS>(c);
        store_rows<BITS>(kc, vc, sub, hmask, p.kc + row[r] * Q::ROW_BYTES, p.vc + row[r] * Q::ROW_BYTES);
        if (sub % (16 / Q::GROUPS) == 0) {
            __nv_bfloat16 *s = p.scale + row[r] * Q::SCALES + group_of<BITS>(sub);
            s[0] = __float2bfloat16(ks);
            s[Q::GROUPS] = __float2bfloat16(vs);
        }
    }
}

__device__ __forceinline__ uint32_t bf2(__nv_bfloat162 x) { return *reinterpret_cast<const uint32_t *>(&x); }
__device__ __forceinline__ __nv_bfloat162 bf2(uint32_t x) { return *reinterpret_cast<const __nv_bfloat162 *>(&x); }

// A lane's eight stored codes -> values.  bf16: code and scale are both bf16 numbers, so one packed product rounds the value
// once; codes become bf16 by bytes and masks (0x4300 | c is 128 + c for c < 128; the sign of an 8-bit code is taken off it).
// float32: the product has at most 15 significant bits and is exact.
template <int BITS> struct Stored;
template <> struct Stored<8> {
    uint2 w;
    __device__ __forceinline__ void load(const unsigned char *row, int sub) { w = __ldcs(reinterpret_cast<const uint2 *>(row + sub * 8)); }
    __device__ __forceinline__ void store(__nv_bfloat16 *out, __nv_bfloat16 scale) const {
        const __nv_bfloat162 s = __halves2bfloat162(scale, scale);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __byte_perm((i < 2 ? w.x : w.y) ^ 0x80808080u, 0x43434343u, i & 1 ? 0x4342 : 0x4140);
            o[i] = bf2(__hmul2(__hsub2(bf2(u & 0xff7fff7fu), bf2(u & 0xff80ff80u)), s));
        }
        *reinterpret_cast<uint4 *>(out) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __device__ __forceinline__ float code(int i) const { return (float)((int)(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 255u) - 128); }
};
template <> struct Stored<4> {
    uint32_t r0, r1;
    __device__ __forceinline__ void load(const unsigned char *row, int sub) {
        const int unit = 8 * (sub & 3) + (sub >> 2);       // runs 2 sub and 2 sub + 1: places 2 (sub % 4), + 1 of the group
        r0 = __ldcs(reinterpret_cast<const unsigned short *>(row + unit * 2));
        r1 = __ldcs(reinterpret_cast<const unsigned short *>(row + unit * 2 + 8));
    }
    __device__ __forceinline__ void store(__nv_bfloat16 *out, __nv_bfloat16 scale) const {
        const __nv_bfloat162 s = __halves2bfloat162(scale, scale), bias = __float2bfloat162_rn(136.f);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = i < 2 ? r0 : r1, two = i & 1 ? (r >> 8) | (r << 4) : r | (r << 12);
            o[i] = bf2(__hmul2(__hsub2(bf2((two & 0x000f000fu) | 0x43004300u), bias), s));
        }
        *reinterpret_cast<uint4 *>(out) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __device__ __forceinline__ float code(int i) const { return (float)((int)(((i < 4 ? r0 : r1) >> (4 * (i & 3))) & 15u) - 8); }
};
template <int BITS>
__device__ __forceinline__ void store_values(float *out, const Stored<BITS> &c, __nv_bfloat16 scale) {
    const float s = __bfloat162float(scale);
    *reinterpret_cast<float4 *>(out) = make_float4(c.code(0) * s, c.code(1) * s, c.code(2) * s, c.code(3) * s);
    *reinterpret_cast<float4 *>(out + 4) = make_float4(c.code(4) * s, c.code(5) * s, c.code(6) * s, c.code(7) * s);
}
template <int BITS>
__device__ __forceinline__ void store_values(__nv_bfloat16 *out, const Stored<BITS> &c, __nv_bfloat16 scale) { c.store(out, scale); }

template <typename T, int BITS>
__global__ void __launch_bounds__(256) quant_read_kernel(const RowsParams p) {
    using Q = Quant<BITS>;
    const int sub = threadIdx.x & 15;
    Stored<BITS> k[AT_ONCE], v[AT_ONCE];
    __nv_bfloat16 ks[AT_ONCE], vs[AT_ONCE];
    T *ko[AT_ONCE], *vo[AT_ONCE];
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {
        const Place w = place_of(p, r);
        ko[r] = nullptr;
        if (!w.any) continue;
        ko[r] = static_cast<T *>(p.k) + w.b * p.kb + w.h * p.kh + w.t * p.kr + sub * 8;
        vo[r] = static_cast<T *>(p.v) + w.b * p.vb + w.h * p.vh + w.t * p.vr + sub * 8;
        const int64_t at = row_position(p, w.b, w.head, w.t);
        if (at < 0) {
            float4 *o[2] = {reinterpret_cast<float4 *>(ko[r]), reinterpret_cast<float4 *>(vo[r])};
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) o[0][i] = o[1][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            ko[r] = nullptr;
            continue;
        }
        const int64_t row = (int64_t)w.head * p.capacity + at;
        k[r].load(p.kc + row * Q::ROW_BYTES, sub);
        v[r].load(p.vc + row * Q::ROW_BYTES, sub);
        const __nv_bfloat16 *s = p.scale + row * Q::SCALES + group_of<BITS>(sub);
        ks[r] = s[0];
        vs[r] = s[Q::GROUPS];
    }
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r)
        if (ko[r]) {
            store_values<BITS>(ko[r], k[r], ks[r]);
            store_values<BITS>(vo[r], v[r], vs[r]);
        }
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
    const float s = group_scale_bf16<BITS>(top);
    const float x[8] = {r.x, r.y, r.z, r.w, 0.f, 0.f, 0.f, 0.f};
    uint32_t c[8];
    stored_codes<BITS, false>(x, s, c);
    constexpr uint32_t MASK = BITS == 8 ? 255u : 15u;
    const uint32_t c0 = c[0] & MASK, c1 = c[1] & MASK, c2 = c[2] & MASK, c3 = c[3] & MASK;
    unsigned char *dst = (is_v ? p.vc : p.kc) + row * Q::ROW_BYTES;
    if (BITS == 8) *reinterpret_cast<uint32_t *>(dst + lane * 4) = c0 | c1 << 8 | c2 << 16 | c3 << 24;
    else *reinterpret_cast<uint16_t *>(dst + ((lane & 7) * 4 + (lane >> 3)) * 2) = (uint16_t)(c0 | c1 << 4 | c2 << 8 | c3 << 12);
    if (lane % (32 / Q::GROUPS) == 0)
        p.scale[row * Q::SCALES + (is_v ? Q::GROUPS : 0) + lane / (32 / Q::GROUPS)] = __float2bfloat16(s);
}

// A flat grid where a CTA would otherwise be mostly idle (a decode step writes one position per sequence).
static dim3 rows_grid(RowsParams &p) {
    p.flat = p.tokens < PER_CTA;
    if (p.flat) return dim3((p.items + PER_CTA - 1) / PER_CTA);
    return dim3((unsigned)(p.tokens + PER_CTA - 1) / PER_CTA, (unsigned)p.h_kv, (unsigned)p.batch);
}

static int rows_check(const skv_qcache *c, const void *k, const void *v, int dtype, int batch, int tokens, int64_t kb,
                      int64_t kh, int64_t kr, int64_t vb, int64_t vh, int64_t vr, const int64_t *pos, int64_t pos0,
                      RowsParams &p) {
    const int rc = qcache_check(c);
    if (rc) return rc;
    if (!k || !v) return SKV_E_NULL;
    if (dtype != SKV_BF16 && dtype != SKV_F32) return SKV_E_DTYPE;
    if (batch <= 0 || batch > c->batch || tokens < 0 || tokens > c->capacity ||
        (int64_t)batch * c->h_kv * tokens > 0x7fffffff)
        return SKV_E_RANGE;
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
    p.items = (uint32_t)batch * c->h_kv * tokens;
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
    const dim3 grid = rows_grid(p);
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
    const dim3 grid = rows_grid(p);
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
