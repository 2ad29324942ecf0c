// The FP8 encoder shared by the weight quantizer (fp8_quant.cu, whose header
// gives the rules and why the hardware converters meet them) and the block
// quantizers (fp8_blocks.cu, block_norm.cu).
#pragma once
#include "common.cuh"
#include "fp8_product.h"

namespace reng {

// Two f32 -> two E4M3 codes (first argument in the low byte).
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t cvt_e5m2x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int FMT>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
    uint32_t c;
    if (FMT == RENG_FP8_E4M3) {
        c = cvt_e4m3x2(fminf(fmaxf(a, -240.0f), 240.0f), fminf(fmaxf(b, -240.0f), 240.0f));
    } else {
        c = cvt_e5m2x2(a, b);
    }
    if (isnan(a)) c = (c & 0xff00u) | ((__float_as_uint(a) >> 24) & 0x80u) | 0x7fu;
    if (isnan(b)) c = (c & 0x00ffu) | ((((__float_as_uint(b) >> 24) & 0x80u) | 0x7fu) << 8);
    return c;
}

// x / s as the reference's host computes it: IEEE division; a NaN weight
// comes through as itself, sign included (x86 returns the NaN operand; GPU
// arithmetic would return its canonical positive NaN), and a NaN generated
// by the division is x86's default NaN, whose sign bit is set.
__device__ __forceinline__ float div_host(float x, float s) {
    if (isnan(x)) return x;
    float q = __fdiv_rn(x, s);
    if (isnan(q)) q = __uint_as_float(0xffc00000u);
    return q;
}

constexpr int kFp8Group = 128;  // columns (and, of a weight block, rows) that share one scale

template <int FMT>
__device__ __forceinline__ float fp8_max_finite() {
    return FMT == RENG_FP8_E4M3 ? 240.0f : 57344.0f;
}

// absmax / max_finite, 1 for a block of zeros.  No lower than the smallest
// normal f32: a quotient that underflowed to 0 would make the block's zeros
// 0 / 0, and a subnormal one has too few bits to divide by.
template <int FMT>
__device__ __forceinline__ float fp8_block_scale(float absmax) {
    return absmax > 0.0f ? fmaxf(__fdiv_rn(absmax, fp8_max_finite<FMT>()), 1.17549435e-38f) : 1.0f;
}

// ------------------------------------------------------------ warp tiles --
// The block operators work on a warp tile: 4 groups of 128 values, 16 values
// per lane.  Two ways to lay a tile over the lanes:
//   VEC      lane l holds columns 16 (l % 8) .. + 15 of group l / 8: wide
//            loads and stores; needs rows on 16 bytes and whole 16-column
//            chunks;
//   not VEC  value e of lane l is column 32 (e % 4) + l of group e / 4: one
//            element per access, consecutive lanes on consecutive elements,
//            for any pitch, alignment and width.
// A group's (row pointer, first column) is the caller's; columns at or past
// `cols` read as 0, which no absmax or sum notices, and are not written.
constexpr int kTileGroups = 4;

// The raw elements of a lane's 16 values.
template <int TYPE, bool VEC>
struct Raw16 {
    static constexpr int N = TYPE == RENG_TYPE_BF16 && VEC ? 8 : 16;
    uint32_t w[N];
};

template <int TYPE, bool VEC>
__device__ __forceinline__ void raw_zero(Raw16<TYPE, VEC>& r) {
#pragma unroll
    for (int i = 0; i < Raw16<TYPE, VEC>::N; i++) r.w[i] = 0u;
}

// Loads go past L1 (each element is read once) unless KEEP, for the vectors
// that every row reads again.
template <bool KEEP, typename T>
__device__ __forceinline__ T ld_elem(const T* p) {
    return KEEP ? *p : __ldcg(p);
}

// VEC: 16 elements from p (16-byte aligned).
template <int TYPE, bool KEEP = false>
__device__ __forceinline__ void raw_load(const void* p, Raw16<TYPE, true>& r) {
#pragma unroll
    for (int i = 0; i < Raw16<TYPE, true>::N / 4; i++) {
        const uint4 q = ld_elem<KEEP>(static_cast<const uint4*>(p) + i);
        r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
    }
}

// not VEC: group g's 4 values of this lane, from column c0 of `row`.
template <int TYPE, bool KEEP = false>
__device__ __forceinline__ void raw_load(const void* row, int64_t c0, int64_t cols, int g, Raw16<TYPE, false>& r) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t c = c0 + 32 * i + lane;
        if (c < cols)
            r.w[4 * g + i] = TYPE == RENG_TYPE_BF16 ? (uint32_t)ld_elem<KEEP>(static_cast<const uint16_t*>(row) + c)
                                                    : ld_elem<KEEP>(static_cast<const uint32_t*>(row) + c);
    }
}

template <int TYPE, bool VEC>
__device__ __forceinline__ void raw_floats(const Raw16<TYPE, VEC>& r, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
        if (TYPE == RENG_TYPE_F32) v[i] = __uint_as_float(r.w[i]);
        else if (VEC) v[i] = (i & 1) ? bf16hi(r.w[i / 2]) : bf16lo(r.w[i / 2]);
        else v[i] = bf16lo(r.w[i]);
    }
}

// Two floats rounded to bf16 (nearest even), the first in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Maximum over a group's lanes of each group's value: VEC has one value per
// lane (8 lanes a group), else 4 values per lane (all lanes).
template <bool VEC>
__device__ __forceinline__ void group_max(uint32_t (&m)[VEC ? 1 : kTileGroups]) {
#pragma unroll
    for (int o = VEC ? 4 : 16; o > 0; o >>= 1)
#pragma unroll
        for (int g = 0; g < (VEC ? 1 : kTileGroups); g++) m[g] = max(m[g], __shfl_xor_sync(0xffffffffu, m[g], o));
}

// The absmax bits of a tile's groups.  Bits of magnitudes order as their
// values do, with NaN above infinity, so one integer maximum also tells
// whether a value is not finite; `odd` says so for the whole warp, and then
// the maximum is taken again without the NaNs.
template <bool VEC>
__device__ __forceinline__ void tile_absmax(const float (&v)[16], uint32_t (&m)[VEC ? 1 : kTileGroups], bool& odd) {
#pragma unroll
    for (int g = 0; g < (VEC ? 1 : kTileGroups); g++) {
        m[g] = 0u;
#pragma unroll
        for (int i = 0; i < (VEC ? 16 : 4); i++) m[g] = max(m[g], abs_bits(v[4 * g + i]));
    }
    uint32_t top = m[0];
#pragma unroll
    for (int g = 1; g < (VEC ? 1 : kTileGroups); g++) top = max(top, m[g]);
    odd = __any_sync(0xffffffffu, top >= 0x7f800000u);
    if (odd) {
#pragma unroll
        for (int g = 0; g < (VEC ? 1 : kTileGroups); g++) {
            m[g] = 0u;
#pragma unroll
            for (int i = 0; i < (VEC ? 16 : 4); i++) {
                const uint32_t a = abs_bits(v[4 * g + i]);
                if (a <= 0x7f800000u) m[g] = max(m[g], a);
            }
        }
    }
}

// Codes of two finite values whose scale holds their block's absmax: the
// quotients are at most max_finite and a rounding, which the converter
// brings back to max_finite, so nothing is clamped and no NaN is looked for.
// r = RN(1 / s); s of at least 2^-60 takes fp8_product.h's correction (the
// correctly rounded quotient), a smaller one the division.
template <int FMT>
__device__ __forceinline__ uint32_t fp8_codes2(float a, float b, float s, float r) {
    const bool product = s >= 8.6736174e-19f;
    const float qa = product ? fp_quotient(a, s, r) : __fdiv_rn(a, s);
    const float qb = product ? fp_quotient(b, s, r) : __fdiv_rn(b, s);
    return FMT == RENG_FP8_E4M3 ? cvt_e4m3x2(qa, qb) : cvt_e5m2x2(qa, qb);
}

// The codes of a lane's 16 values, 4 to a word in order, given the scale of
// each of its groups.
template <int FMT, bool VEC>
__device__ __forceinline__ uint4 tile_codes(const float (&v)[16], const float (&s)[VEC ? 1 : kTileGroups], bool odd) {
    uint32_t w[4];
    if (odd) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float sc = s[VEC ? 0 : i];
            w[i] = encode2<FMT>(div_host(v[4 * i], sc), div_host(v[4 * i + 1], sc)) |
                   encode2<FMT>(div_host(v[4 * i + 2], sc), div_host(v[4 * i + 3], sc)) << 16;
        }
    } else {
        float r[VEC ? 1 : kTileGroups];
#pragma unroll
        for (int g = 0; g < (VEC ? 1 : kTileGroups); g++) r[g] = __frcp_rn(s[g]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float sc = s[VEC ? 0 : i], rc = r[VEC ? 0 : i];
            w[i] = fp8_codes2<FMT>(v[4 * i], v[4 * i + 1], sc, rc) |
                   fp8_codes2<FMT>(v[4 * i + 2], v[4 * i + 3], sc, rc) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// not VEC: group g's 4 codes of this lane.
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t c0, int64_t cols, uint32_t codes) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t c = c0 + 32 * i + lane;
        if (c < cols) row[c] = (uint8_t)(codes >> (8 * i));
    }
}

}  // namespace reng
