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

// The running absmax of |x|: '>' against it, so a NaN is never taken.
__device__ __forceinline__ float fp8_absmax(float m, float x) {
    const float a = fabsf(x);
    return a > m ? a : m;
}

// absmax / max_finite, 1 for a block of zeros.  No lower than the smallest
// normal f32: a quotient that underflowed to 0 would make the block's zeros
// 0 / 0, and a subnormal one has too few bits to divide by.
template <int FMT>
__device__ __forceinline__ float fp8_block_scale(float absmax) {
    return absmax > 0.0f ? fmaxf(__fdiv_rn(absmax, fp8_max_finite<FMT>()), 1.17549435e-38f) : 1.0f;
}

// encode(v[i] / s) of 8 values whose magnitudes are at most absmax, the
// quotients by fp8_product.h's correction where it admits the scale and by
// the division elsewhere.  fp_quotient keeps a NaN's sign; an infinity makes
// s infinite, so its block takes the division.
template <int FMT>
__device__ __forceinline__ uint2 fp8_encode8(const float (&v)[8], float s, float absmax) {
    uint32_t c[4];
    const float r = __frcp_rn(s);
    if (fp8_product_ok(s, r, absmax)) {
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = encode2<FMT>(fp_quotient(v[2 * i], s, r), fp_quotient(v[2 * i + 1], s, r));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = encode2<FMT>(div_host(v[2 * i], s), div_host(v[2 * i + 1], s));
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// Maximum over the 16 lanes of a half-warp (one 128-value group).
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// -------------------------------------------------- 8 consecutive values --
// Loads and stores of 8 consecutive elements at column c of a row of `cols`.
// VEC: rows and base are 16-byte aligned (8 for codes) and the 8 elements
// take one or two wide accesses where they all exist; the row's last partial
// chunk, and every chunk without VEC, goes element by element.  Columns past
// the end read as 0, which no absmax or sum notices, and are not written.
template <int TYPE, bool VEC>
__device__ __forceinline__ void load8(const void* row, int64_t c, int64_t cols, float (&v)[8]) {
    if (VEC && c + 8 <= cols) {
        if (TYPE == RENG_TYPE_BF16) {
            const uint4 u = ldg_stream(static_cast<const uint16_t*>(row) + c);
            v[0] = bf16lo(u.x), v[1] = bf16hi(u.x), v[2] = bf16lo(u.y), v[3] = bf16hi(u.y);
            v[4] = bf16lo(u.z), v[5] = bf16hi(u.z), v[6] = bf16lo(u.w), v[7] = bf16hi(u.w);
        } else {
            const uint4 a = ldg_stream(static_cast<const float*>(row) + c);
            const uint4 b = ldg_stream(static_cast<const float*>(row) + c + 4);
            v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z);
            v[3] = __uint_as_float(a.w), v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y);
            v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = 0.f;
        if (c + i < cols)
            v[i] = TYPE == RENG_TYPE_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(row)[c + i])
                                          : static_cast<const float*>(row)[c + i];
    }
}

template <bool VEC>
__device__ __forceinline__ void store_codes8(uint8_t* row, int64_t c, int64_t cols, uint2 q) {
    if (VEC && c + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + c) = q;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (c + i < cols) row[c + i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}

}  // namespace reng
