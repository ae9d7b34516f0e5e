// The quantised form of a cached row (128 values of one token of one KV head) and the device functions that make it and
// read it.  BITS 8: one scale per row, codes in order.  BITS 4: one scale for each 32 values; two codes per byte, the
// lower nibble first, and the row's 32 runs of four values stored in the order (run % 8, run / 8): the 8 bytes a lane
// reads then hold one run of each scale group at the same place for every lane, which is what the matrix products of
// the attention need (one scale per product, not one per lane).
//   scale = bf16(max |x| / MOST), code = round(x / scale) within +-MOST, stored with BIAS added
// The scale is rounded to bf16 before the codes are taken, so its rounding costs no accuracy: |x - code * scale| is at
// most scale / 2 (the largest value's quotient is at most MOST (1 + 2^-8), within half a step of MOST).
// Groups whose scale is below the smallest normal number are stored as zeros; a group that holds an Inf or NaN has a NaN
// scale and reads back as NaN.
#pragma once

#include "skv_common.cuh"

namespace skv {

template <int BITS>
struct Quant {
    static_assert(BITS == 8 || BITS == 4, "8 or 4 bits");
    static constexpr int GROUPS = BITS == 8 ? 1 : 4;       // scales per row
    static constexpr int MOST = BITS == 8 ? 127 : 7;       // largest code
    static constexpr int BIAS = BITS == 8 ? 128 : 8;
    static constexpr int ROW_BYTES = HEAD_DIM * BITS / 8;
    static constexpr int SCALES = 2 * GROUPS;              // per cached position: the key's, then the value's
};

// Magnitude bits of a float: ordered like the magnitudes, with Inf above every number and NaN above Inf.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int BITS>
__device__ __forceinline__ float group_scale(uint32_t largest) {
    if (largest >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const float s = __bfloat162float(__float2bfloat16(__fdiv_rn(__uint_as_float(largest), (float)Quant<BITS>::MOST)));
    return s < 1.17549435e-38f ? 0.f : s;
}

// An IEEE quotient: for a bf16 value and a bf16 scale it is exact wherever the true quotient lies half-way between two
// codes and far enough from there otherwise, so the code is the nearest one (ties to even) of the true quotient.
template <int BITS>
__device__ __forceinline__ uint32_t stored_code(float x, float scale) {
    constexpr float M = (float)Quant<BITS>::MOST;
    const float c = scale > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -M), M) : 0.f;
    return (uint32_t)((int)c + Quant<BITS>::BIAS);
}

// Eight consecutive values (lane `sub` of 16 owns components 8 sub .. 8 sub + 7) -> their place in the stored row.
// The lanes of a half warp call this together.  Returns the scale of the lane's group.
template <int BITS>
__device__ __forceinline__ float quantise_row8(const float (&x)[8], int sub, unsigned hmask, unsigned char *row,
                                               bool store) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(x[i]));
#pragma unroll
    for (int o = 1; o < (BITS == 8 ? 16 : 4); o <<= 1) top = max(top, __shfl_xor_sync(hmask, top, o, 16));
    const float s = group_scale<BITS>(top);
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = stored_code<BITS>(x[i], s);
    if (BITS == 8) {
        uint2 w;
        w.x = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        w.y = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
        if (store) *reinterpret_cast<uint2 *>(row + sub * 8) = w;
    } else {
        // runs 2 sub and 2 sub + 1: group sub / 4, places j = 2 (sub % 4) and j + 1; the neighbouring group's lane
        // (sub ^ 4) has the run that lies beside either of them
        const uint32_t r0 = c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12, r1 = c[4] | c[5] << 4 | c[6] << 8 | c[7] << 12;
        const int grp = sub >> 2, j = 2 * (sub & 3);
        const bool odd = grp & 1;
        const uint32_t other = __shfl_xor_sync(hmask, odd ? r0 : r1, 4, 16);
        const uint32_t w = odd ? (other | r1 << 16) : (r0 | other << 16);
        const int unit = odd ? (j + 1) * 4 + grp - 1 : j * 4 + grp;
        if (store) *reinterpret_cast<uint32_t *>(row + unit * 2) = w;
    }
    return s;
}

// The inverse: the lane's eight values of a stored row, given the scale of the lane's group.
template <int BITS>
__device__ __forceinline__ void restore_row8(const unsigned char *row, int sub, float scale, float (&x)[8]) {
    if (BITS == 8) {
        const uint2 w = *reinterpret_cast<const uint2 *>(row + sub * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = (float)((int)((w.x >> (8 * i)) & 255u) - 128) * scale;
            x[4 + i] = (float)((int)((w.y >> (8 * i)) & 255u) - 128) * scale;
        }
    } else {
        const int grp = sub >> 2, j = 2 * (sub & 3);
        const uint32_t r0 = *reinterpret_cast<const uint16_t *>(row + (j * 4 + grp) * 2);
        const uint32_t r1 = *reinterpret_cast<const uint16_t *>(row + (j * 4 + 4 + grp) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = (float)((int)((r0 >> (4 * i)) & 15u) - 8) * scale;
            x[4 + i] = (float)((int)((r1 >> (4 * i)) & 15u) - 8) * scale;
        }
    }
}

// Scale group of the eight values lane `sub` owns.
template <int BITS>
__device__ __forceinline__ int group_of(int sub) { return BITS == 8 ? 0 : sub >> 2; }

// Host-side checks shared by every entry point that takes a quantised cache (no CUDA call).
static inline int qcache_check(const skv_qcache *c) {
    if (!c || !c->k || !c->v || !c->scale) return SKV_E_NULL;
    if (c->d != HEAD_DIM) return SKV_E_DIM;
    if (c->bits != 8 && c->bits != 4) return SKV_E_RANGE;
    if (c->batch <= 0 || c->h_kv <= 0 || c->capacity <= 0 || (int64_t)c->batch * c->h_kv > 65535) return SKV_E_RANGE;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->scale)) return SKV_E_ALIGN;
    return SKV_OK;
}

}  // namespace skv
