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

// The stored codes of eight values, as the low bits of the results.  Adding 1.5 * 2^23 rounds a quotient to an integer, ties
// to even, and leaves it, biased, in the low bits; no clamp is needed, since the scale is at most 2^-9 of itself too small.
// EXACT: an IEEE quotient.  Else the values are bf16, like the scale: a quotient from the rounded reciprocal y with one
// correction by its exact remainder (Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).
// Where the true quotient lies half-way between two codes it is a float32 number t, the first quotient is t + d, its
// remainder -s d, and the corrected one t - d (1 - s y) rounds to t; everywhere else two 8-bit significands keep the
// quotient 2^-16 of itself away from there.  So the code is the nearest one (ties to even) of the true quotient.
// (Remainders of scales below 2^-90 could leave the numbers: those take the IEEE quotient as well.)
template <int BITS, bool EXACT>
__device__ __forceinline__ void stored_codes(const float (&x)[8], float scale, uint32_t (&c)[8]) {
    constexpr float ROUND = 12582912.f + (float)Quant<BITS>::BIAS;
    if (!(scale > 0.f)) {                                  // zeros, or a group that has no scale
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = Quant<BITS>::BIAS;
    } else if (EXACT || scale < 8.077936e-28f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(__fdiv_rn(x[i], scale) + ROUND);
    } else {
        const float y = __frcp_rn(scale);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = x[i] * y;
            c[i] = __float_as_uint(fmaf(fmaf(-q, scale, x[i]), y, q) + ROUND);
        }
    }
}

// Eight consecutive values (lane `sub` of 16 owns components 8 sub .. 8 sub + 7), whose largest magnitude has the bits
// `top`, -> their place in the stored row.  The lanes of a half warp call this together.  Returns the lane's group's scale.
template <int BITS, bool EXACT>
__device__ __forceinline__ float quantise_row8(const float (&x)[8], uint32_t top, int sub, unsigned hmask,
                                               unsigned char *row) {
#pragma unroll
    for (int o = 1; o < (BITS == 8 ? 16 : 4); o <<= 1) top = max(top, __shfl_xor_sync(hmask, top, o, 16));
    const float s = group_scale<BITS>(top);
    uint32_t c[8];
    stored_codes<BITS, EXACT>(x, s, c);
    if (BITS == 8) {
        uint2 w;
        w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2 *>(row + sub * 8) = w;
    } else {
        // runs 2 sub and 2 sub + 1: group sub / 4, places j = 2 (sub % 4) and j + 1; the neighbouring group's lane
        // (sub ^ 4) has the run that lies beside either of them
        const uint32_t r0 = (c[0] & 15u) | (c[1] & 15u) << 4 | (c[2] & 15u) << 8 | (c[3] & 15u) << 12;
        const uint32_t r1 = (c[4] & 15u) | (c[5] & 15u) << 4 | (c[6] & 15u) << 8 | (c[7] & 15u) << 12;
        const int grp = sub >> 2, j = 2 * (sub & 3);
        const bool odd = grp & 1;
        const uint32_t other = __shfl_xor_sync(hmask, odd ? r0 : r1, 4, 16);
        const uint32_t w = odd ? (other | r1 << 16) : (r0 | other << 16);
        const int unit = odd ? (j + 1) * 4 + grp - 1 : j * 4 + grp;
        *reinterpret_cast<uint32_t *>(row + unit * 2) = w;
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
