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
#include "skv_pairs.cuh"

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

// The same for values that are bf16 themselves (`largest`: the float32 bits of one).  The quotient by 127 or 7 of an 8-bit
// significand stays 2^-16 of itself away from the middle between two bf16 numbers, so a product with the rounded 1 / 127 or
// 1 / 7 rounds to the same scale.
template <int BITS>
__device__ __forceinline__ float group_scale_bf16(uint32_t largest) {
    const float s = __bfloat162float(__float2bfloat16(__uint_as_float(largest) * (1.f / (float)Quant<BITS>::MOST)));
    return largest >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : s < 1.17549435e-38f ? 0.f : s;
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The stored codes of eight values, as the low bits of the results.  Adding 1.5 * 2^23 rounds a quotient to an integer, ties
// to even, and leaves it, biased, in the low bits; no clamp is needed, since the scale is at most 2^-8 of itself too small.
// EXACT: an IEEE quotient.  Else the values are bf16, like the scale: a quotient from a reciprocal y with one correction by
// its exact remainder (Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).  Where the true
// quotient lies half-way between two codes it is a float32 number t, the first quotient is t + d, its remainder -s d, and the
// corrected one t + d (1 - s y) rounds to t; everywhere else two 8-bit significands keep the quotient 2^-16 of itself away
// from there.  So the code is the nearest one (ties to even) of the true quotient, with a reciprocal good to 2^-22.
// (Remainders of scales below 2^-90 could leave the numbers: those take the IEEE quotient as well.)
template <int BITS, bool EXACT>
__device__ __forceinline__ void stored_codes(const float (&x)[8], float scale, uint32_t (&c)[8]) {
    constexpr float ROUND = 12582912.f + (float)Quant<BITS>::BIAS;
    if (!EXACT && scale >= 8.077936e-28f) {
        const float y = rcp_approx(scale);
        const float2 y2 = make_float2(y, y), s2 = make_float2(-scale, -scale), round = make_float2(ROUND, ROUND);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 v = make_float2(x[i], x[i + 1]), q = mul2(v, y2);
            const float2 t = add2(fma2(fma2(q, s2, v), y2, q), round);
            c[i] = __float_as_uint(t.x);
            c[i + 1] = __float_as_uint(t.y);
        }
    } else {
        const bool some = scale > 0.f;                     // else zeros, or a group that has no scale
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = __float_as_uint((some ? __fdiv_rn(x[i], scale) : 0.f) + ROUND);
    }
}

// Eight codes -> the lane's bytes of the stored row: 8 bits: eight bytes in order; 4 bits: the two runs (lower 16 bits of each).
template <int BITS>
__device__ __forceinline__ uint2 packed_codes(const uint32_t (&c)[8]) {
    if (BITS == 8)
        return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                          __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
    // (above a code lies 0x4b4000, whose low bits are zero: sums of shifted codes carry nothing into the lower 16)
    return make_uint2(((c[3] << 4) + c[2] << 8) + ((c[1] << 4) + c[0]), ((c[7] << 4) + c[6] << 8) + ((c[5] << 4) + c[4]));
}

// Key and value of a position, lane `sub` of 16 with its eight codes of each (packed_codes), into their stored rows.  4 bits:
// the lane's runs 2 sub and 2 sub + 1 belong to group sub / 4, places j = 2 (sub % 4) and j + 1; the neighbouring group's
// lane (sub ^ 4) has the run that lies beside either of them: one exchange for key and value.
template <int BITS>
__device__ __forceinline__ void store_rows(uint2 k, uint2 v, int sub, unsigned hmask, unsigned char *krow, unsigned char *vrow) {
    if (BITS == 8) {
        *reinterpret_cast<uint2 *>(krow + sub * 8) = k;
        *reinterpret_cast<uint2 *>(vrow + sub * 8) = v;
    } else {
        const bool odd = (sub >> 2) & 1;
        const uint32_t other = __shfl_xor_sync(hmask, odd ? __byte_perm(k.x, v.x, 0x5410) : __byte_perm(k.y, v.y, 0x5410), 4, 16);
        const int unit = odd ? 8 * (sub & 3) + 4 + (sub >> 2) - 1 : 8 * (sub & 3) + (sub >> 2);
        *reinterpret_cast<uint32_t *>(krow + unit * 2) = odd ? __byte_perm(other, k.y, 0x5410) : __byte_perm(k.x, other, 0x5410);
        *reinterpret_cast<uint32_t *>(vrow + unit * 2) = odd ? __byte_perm(other, v.y, 0x5432) : __byte_perm(v.x, other, 0x7610);
    }
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
    if (c->batch <= 0 || c->skip < 0 || c->h_kv <= 0 || c->capacity <= 0 ||
        ((int64_t)c->skip + c->batch) * c->h_kv > 65535)
        return SKV_E_RANGE;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->scale)) return SKV_E_ALIGN;
    return SKV_OK;
}

// Where the rows of the struct's sequences begin.  (The scales may begin on any position's: no load of them takes more than one
// position's, 4 bytes in 8 bits and 16 in 4.)
struct QuantRows {
    unsigned char *k, *v;
    __nv_bfloat16 *scale;
    int32_t *status;
};
static inline QuantRows qcache_rows(const skv_qcache *c) {
    const int64_t heads = (int64_t)c->skip * c->h_kv, rows = heads * c->capacity, codes = rows * (HEAD_DIM * c->bits / 8);
    return {static_cast<unsigned char *>(c->k) + codes, static_cast<unsigned char *>(c->v) + codes,
            static_cast<__nv_bfloat16 *>(c->scale) + rows * (c->bits == 8 ? Quant<8>::SCALES : Quant<4>::SCALES),
            c->status ? c->status + heads : nullptr};
}

}  // namespace skv
