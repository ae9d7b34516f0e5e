// Writing rows into a quantised KV cache and reading them back.
//
// A prefill chunk is bounded by the memory, with the instructions close behind (eight sequences x 8 heads x 2,048 positions in
// 4 bits, under a profiler: write 23 us for 86 MB, 65 % of the issue slots taken; read 15.4 us); a decode step's few rows by
// the launch.  An IEEE division per value made the write 35 us.
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
};

constexpr int AT_ONCE = 2;       // positions of a half warp in a chunk

// Cache row of a call's first token of sequence `b` (-1 - capacity: none of its rows lies in the cache).
__device__ __forceinline__ int64_t first_row(const RowsParams &p, int b) {
    const int64_t first = p.pos ? p.pos[p.pos_per_seq ? b : 0] : p.pos0;
    return first < 0 || first > p.capacity ? -1 - (int64_t)p.capacity : first;
}
// The row as an index; -1 (recorded in the head's status) where it lies outside the cache.
__device__ __forceinline__ int cache_row(const RowsParams &p, int head, int64_t at) {
    if (at >= 0 && at < p.capacity) return (int)at;
    if (p.status) atomicOr(p.status + head, SKV_ST_BAD_INDEX);
    return -1;
}

// The positions of a half warp.  A chunk: 3-d grid (positions, KV heads, sequences), N positions 16 apart, so that only the
// first one's addresses are computed.  FLAT, for few tokens per sequence: one position of a flat grid over all.
template <bool FLAT>
struct Places {
    static constexpr int N = FLAT ? 1 : AT_ONCE;
    int b, h, t, head, count;    // first token; positions there are
    int64_t first;               // cache row of token 0
    __device__ __forceinline__ explicit Places(const RowsParams &p) {
        const int half = threadIdx.x >> 4;
        if (FLAT) {
            const uint32_t item = blockIdx.x * 16 + half;
            head = (int)(item / (uint32_t)p.tokens);
            t = (int)(item - (uint32_t)head * p.tokens);
            b = head / p.h_kv;
            h = head - b * p.h_kv;
            count = item < p.items;
        } else {
            t = (int)blockIdx.x * (16 * N) + half;
            h = blockIdx.y;
            b = blockIdx.z;
            head = b * p.h_kv + h;
            count = t < p.tokens ? min(N, (p.tokens - t + 15) >> 4) : 0;
        }
        if (!count) b = h = head = t = 0;
        first = first_row(p, b);
    }
    // cache row of the r-th position
    __device__ __forceinline__ int row(const RowsParams &p, int r) const { return cache_row(p, head, first + t + 16 * r); }
};

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

template <typename T, int BITS, bool FLAT>
__global__ void __launch_bounds__(256) quant_write_kernel(const RowsParams p) {
    using Q = Quant<BITS>;
    constexpr bool EXACT = sizeof(T) == 4;
    pdl_wait();
    pdl_trigger();
    const int sub = threadIdx.x & 15;
    const unsigned hmask = (threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu;
    const Places<FLAT> w(p);                               // (everything about a position is uniform within its half warp)
    constexpr int N = Places<FLAT>::N;
    const T *kg = static_cast<const T *>(p.k) + (w.b * p.kb + w.h * p.kh + w.t * p.kr + sub * 8);
    const T *vg = static_cast<const T *>(p.v) + (w.b * p.vb + w.h * p.vh + w.t * p.vr + sub * 8);
    Eight<T> k[N], v[N];
    int row[N];
#pragma unroll
    for (int r = 0; r < N; ++r, kg += 16 * p.kr, vg += 16 * p.vr) {
        row[r] = r < w.count ? w.row(p, r) : -1;
        if (row[r] < 0) continue;
        k[r].load(kg);
        v[r].load(vg);
    }
    const int64_t base = (int64_t)w.head * p.capacity;
    unsigned char *const kc = p.kc + base * Q::ROW_BYTES, *const vc = p.vc + base * Q::ROW_BYTES;
    __nv_bfloat16 *const scale = p.scale + base * Q::SCALES + group_of<BITS>(sub);
#pragma unroll
    for (int r = 0; r < N; ++r) {
        if (row[r] < 0) continue;
        float ks, vs, x[8];
        uint32_t c[8];
        scales_of<BITS>(k[r], v[r], hmask, ks, vs);
        k[r].values(x);
        stored_codes<BITS, EXACT>(x, ks, c);
        const uint2 kp = packed_codes<BITS>(c);
        v[r].values(x);
        stored_codes<BITS, EXACT>(x, vs, c);
        const uint2 vp = packed_codes<BITS>(c);
        store_rows<BITS>(kp, vp, sub, hmask, kc + (int64_t)row[r] * Q::ROW_BYTES, vc + (int64_t)row[r] * Q::ROW_BYTES);
        if (sub % (16 / Q::GROUPS) == 0) {
            __nv_bfloat16 *s = scale + (int64_t)row[r] * Q::SCALES;
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
    __device__ __forceinline__ void load(const unsigned char *row, int sub) {
        w = __ldcs(reinterpret_cast<const uint2 *>(row + sub * 8));
    }
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
    __device__ __forceinline__ float code(int i) const {
        return (float)((int)(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 255u) - 128);
    }
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
    __device__ __forceinline__ float code(int i) const {
        return (float)((int)(((i < 4 ? r0 : r1) >> (4 * (i & 3))) & 15u) - 8);
    }
};
template <int BITS>
__device__ __forceinline__ void store_values(float *out, const Stored<BITS> &c, __nv_bfloat16 scale) {
    const float s = __bfloat162float(scale);
    *reinterpret_cast<float4 *>(out) = make_float4(c.code(0) * s, c.code(1) * s, c.code(2) * s, c.code(3) * s);
    *reinterpret_cast<float4 *>(out + 4) = make_float4(c.code(4) * s, c.code(5) * s, c.code(6) * s, c.code(7) * s);
}
template <int BITS>
__device__ __forceinline__ void store_values(__nv_bfloat16 *out, const Stored<BITS> &c, __nv_bfloat16 scale) {
    c.store(out, scale);
}

template <typename T, int BITS, bool FLAT>
__global__ void __launch_bounds__(256) quant_read_kernel(const RowsParams p) {
    using Q = Quant<BITS>;
    pdl_wait();
    pdl_trigger();
    const int sub = threadIdx.x & 15;
    const Places<FLAT> w(p);
    constexpr int N = Places<FLAT>::N;
    const int64_t base = (int64_t)w.head * p.capacity;
    const unsigned char *const kc = p.kc + base * Q::ROW_BYTES, *const vc = p.vc + base * Q::ROW_BYTES;
    const __nv_bfloat16 *const scale = p.scale + base * Q::SCALES + group_of<BITS>(sub);
    Stored<BITS> k[N], v[N];
    __nv_bfloat16 ks[N], vs[N];
    int row[N];
#pragma unroll
    for (int r = 0; r < N; ++r) {
        row[r] = r < w.count ? w.row(p, r) : -1;
        if (row[r] < 0) continue;
        k[r].load(kc + (int64_t)row[r] * Q::ROW_BYTES, sub);
        v[r].load(vc + (int64_t)row[r] * Q::ROW_BYTES, sub);
        const __nv_bfloat16 *s = scale + (int64_t)row[r] * Q::SCALES;
        ks[r] = s[0];
        vs[r] = s[Q::GROUPS];
    }
    T *kg = static_cast<T *>(p.k) + (w.b * p.kb + w.h * p.kh + w.t * p.kr + sub * 8);
    T *vg = static_cast<T *>(p.v) + (w.b * p.vb + w.h * p.vh + w.t * p.vr + sub * 8);
#pragma unroll
    for (int r = 0; r < N; ++r, kg += 16 * p.kr, vg += 16 * p.vr) {
        if (r >= w.count) continue;
        if (row[r] >= 0) {
            store_values<BITS>(kg, k[r], ks[r]);
            store_values<BITS>(vg, v[r], vs[r]);
        } else {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<float4 *>(kg)[i] = reinterpret_cast<float4 *>(vg)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
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
    const int64_t pos = cache_row(p, head, first_row(p, b));
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

// A flat grid where a chunk's CTA would be mostly idle (a decode step writes one position per sequence).
static bool rows_flat(const RowsParams &p) { return p.tokens < 16 * AT_ONCE; }
static dim3 rows_grid(const RowsParams &p) {
    if (rows_flat(p)) return dim3((p.items + 15) / 16);
    return dim3((unsigned)(p.tokens + 16 * AT_ONCE - 1) / (16 * AT_ONCE), (unsigned)p.h_kv, (unsigned)p.batch);
}
template <typename T, int BITS>
static cudaError_t launch_write(const RowsParams &p, cudaStream_t st) {
    auto kern = rows_flat(p) ? quant_write_kernel<T, BITS, true> : quant_write_kernel<T, BITS, false>;
    return launch_early(kern, rows_grid(p), dim3(256), 0, st, p);
}
template <typename T, int BITS>
static cudaError_t launch_read(const RowsParams &p, cudaStream_t st) {
    auto kern = rows_flat(p) ? quant_read_kernel<T, BITS, true> : quant_read_kernel<T, BITS, false>;
    return launch_early(kern, rows_grid(p), dim3(256), 0, st, p);
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
    const QuantRows at = qcache_rows(c);
    p.kc = at.k; p.vc = at.v; p.scale = at.scale; p.status = at.status;
    p.pos = pos; p.pos0 = pos0;
    p.batch = batch; p.h_kv = c->h_kv; p.capacity = c->capacity; p.tokens = tokens;
    p.items = (uint32_t)batch * c->h_kv * tokens;
    return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int skv_quant_write(const skv_qcache *c, const skv_rows *r, void *stream) {
    if (!r) return SKV_E_NULL;
    RowsParams p;
    const int rc = rows_check(c, r->k, r->v, r->dtype, r->batch, r->tokens, r->k_batch_stride, r->k_head_stride, r->k_row_stride,
                              r->v_batch_stride, r->v_head_stride, r->v_row_stride, r->pos, r->pos0, p);
    if (rc) return rc;
    if (r->tokens == 0) return SKV_OK;
    p.pos_per_seq = r->pos_per_seq;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = r->dtype == SKV_BF16;
    if (c->bits == 8) SKV_CUDA_OK((bf16 ? launch_write<__nv_bfloat16, 8>(p, st) : launch_write<float, 8>(p, st)));
    else SKV_CUDA_OK((bf16 ? launch_write<__nv_bfloat16, 4>(p, st) : launch_write<float, 4>(p, st)));
    SKV_CUDA_OK(cudaGetLastError());
    return SKV_OK;
}

extern "C" int skv_quant_read(const skv_qcache *c, const skv_rows *r, void *stream) {
    if (!r) return SKV_E_NULL;
    RowsParams p;
    const int rc = rows_check(c, r->k, r->v, r->dtype, r->batch, r->tokens, r->k_batch_stride, r->k_head_stride, r->k_row_stride,
                              r->v_batch_stride, r->v_head_stride, r->v_row_stride, r->pos, r->pos0, p);
    if (rc) return rc;
    if (r->tokens == 0) return SKV_OK;
    p.pos_per_seq = r->pos_per_seq;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = r->dtype == SKV_BF16;
    if (c->bits == 8) SKV_CUDA_OK((bf16 ? launch_read<__nv_bfloat16, 8>(p, st) : launch_read<float, 8>(p, st)));
    else SKV_CUDA_OK((bf16 ? launch_read<__nv_bfloat16, 4>(p, st) : launch_read<float, 4>(p, st)));
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
