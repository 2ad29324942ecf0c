// The FP8 encoder shared by the weight quantizer (fp8_quant.cu, whose header
// gives the rules and why the hardware converters meet them) and the block
// quantizers (fp8_blocks.cu, block_norm.cu).
#pragma once
#include <type_traits>

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

// absmax / max_finite, 1 for a block of zeros: the correctly rounded quotient
// by fp8_product.h's correction (checked for both constants over every
// mantissa), an infinite absmax as itself.  No lower than the smallest normal
// f32: a quotient that underflowed to 0 would make the block's zeros 0 / 0,
// and a subnormal one has too few bits to divide by.
template <int FMT>
__device__ __forceinline__ float fp8_block_scale(float absmax) {
    constexpr float d = FMT == RENG_FP8_E4M3 ? 240.0f : 57344.0f, r = 1.0f / d;
    const float y = __fmul_rn(absmax, r), q = __fmaf_rn(__fmaf_rn(-y, d, absmax), r, y);
    const float s = absmax < __int_as_float(0x7f800000) ? fmaxf(q, 1.17549435e-38f) : absmax;
    return absmax > 0.0f ? s : 1.0f;
}

// ------------------------------------------------------------ warp tiles --
// The block operators work on a warp tile: 4 groups of 128 values, 16 values
// per lane, in G groups of the lane's own.  Three ways to lay it out:
//   G 1  lane l holds columns 16 (l % 8) .. + 15 of group l / 8: the fewest
//        scales and shuffles, 32 bytes of a bf16 row a lane (the quantizers);
//   G 2  columns 8 (l % 16) .. + 7 of groups l / 16 and 2 + l / 16:
//        consecutive lanes on consecutive 16 bytes of a bf16 row and 32 of an
//        f32 one (the norm, whose shared memory takes no bank conflicts then,
//        and quantizers of rows of whole 8-column pieces);
//   G 4  columns l, 32 + l, 64 + l and 96 + l of every group: one element per
//        access, consecutive lanes on consecutive elements, for any pitch,
//        alignment and width.
// Columns are below 2^31.  G 1 and 2 need rows on 16 bytes and whole 16- or
// 8-column pieces.  A group's (row pointer, first column) is the caller's;
// columns at or past `cols` read as 0, which no absmax or sum notices, and are
// not written.
constexpr int kTileGroups = 4;
// This lane's group of index g among the tile's 4, and its first column there.
template <int G>
__device__ __forceinline__ int lane_group(int g) {
    const int lane = threadIdx.x & 31;
    return G == 1 ? lane >> 3 : G == 2 ? 2 * g + (lane >> 4) : g;
}
template <int G>
__device__ __forceinline__ int lane_col() {
    const int lane = threadIdx.x & 31;
    return G == 1 ? (lane & 7) * 16 : G == 2 ? (lane & 15) * 8 : 0;
}
// Whether this lane writes its groups' scales.
template <int G>
__device__ __forceinline__ bool lane_first() {
    return (threadIdx.x & (8 * G - 1)) == 0;
}

// The raw elements of a lane's 16 values, group by group.
template <int TYPE, int G>
struct Raw16 {
    static constexpr int N = TYPE == RENG_TYPE_BF16 && G < 4 ? 8 : 16;
    uint32_t w[N];
};

template <int TYPE, int G>
__device__ __forceinline__ void raw_zero(Raw16<TYPE, G>& r) {
#pragma unroll
    for (int i = 0; i < Raw16<TYPE, G>::N; i++) r.w[i] = 0u;
}

// Loads go past L1 (each element is read once) unless KEEP, for the vectors
// that every row reads again.
template <bool KEEP, typename T>
__device__ __forceinline__ T ld_elem(const T* p) {
    return KEEP ? *p : __ldcg(p);
}

// G 1, 2: group g's values of this lane, from p (16-byte aligned).
template <int TYPE, bool KEEP = false, int G>
__device__ __forceinline__ void raw_load(const void* p, int g, Raw16<TYPE, G>& r) {
    constexpr int n = Raw16<TYPE, G>::N / (4 * G);  // 16-byte loads
#pragma unroll
    for (int i = 0; i < n; i++) {
        const uint4 q = ld_elem<KEEP>(static_cast<const uint4*>(p) + i);
        const int k = 4 * (n * g + i);
        r.w[k] = q.x, r.w[k + 1] = q.y, r.w[k + 2] = q.z, r.w[k + 3] = q.w;
    }
}

// G 4: group g's 4 values of this lane, from column c0 of `row`.  WHOLE: the
// group lies inside the row, no element is tested (a whole warp's case, half
// the instructions; callers take all loads of a warp one way or the other, so
// that none waits behind a branch).
template <int TYPE, bool KEEP = false, bool WHOLE = false>
__device__ __forceinline__ void raw_load(const void* row, int c0, int cols, int g, Raw16<TYPE, 4>& r) {
    using E = std::conditional_t<TYPE == RENG_TYPE_BF16, uint16_t, uint32_t>;
    const int c = c0 + (threadIdx.x & 31);
    const E* p = static_cast<const E*>(row) + c;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (WHOLE || c + 32 * i < cols) r.w[4 * g + i] = (uint32_t)ld_elem<KEEP>(p + 32 * i);
}

// A lane's values are handled two at a time: one instruction on a register
// pair, which these kernels' arithmetic needs (with it they still fill 57 to 68%
// of the issue slots while HBM streams).
typedef unsigned long long f2;
__device__ __forceinline__ f2 make_f2(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f2 make_f2(float v) { return make_f2(v, v); }
__device__ __forceinline__ void split_f2(f2 v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f2 mul_f2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add_f2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma_f2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template <int TYPE, int G>
__device__ __forceinline__ void raw_floats(const Raw16<TYPE, G>& r, f2 (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (TYPE == RENG_TYPE_F32) v[i] = make_f2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
        else if (G < 4) v[i] = make_f2(bf16lo(r.w[i]), bf16hi(r.w[i]));
        else v[i] = make_f2(bf16lo(r.w[2 * i]), bf16lo(r.w[2 * i + 1]));
    }
}

// Two floats rounded to bf16 (nearest even), the first in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// max(m, |x|, |y|), NaN if x or y is.
__device__ __forceinline__ float absmax_nan(float m, float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(x)), "f"(fabsf(y)));
    return r;
}

// Maximum over a group's lanes (8 G of them): a lane's is that of its group
// lane % G.  Where a lane holds several groups it hands away half of them at a
// step, so four groups take 6 shuffles and not 20.
template <int G>
__device__ __forceinline__ float group_max(const float (&m)[G]) {
    const bool b0 = threadIdx.x & 1, b1 = threadIdx.x & 2;
    auto merge = [](bool upper, float lo, float hi, int o) {
        return fmaxf(upper ? hi : lo, __shfl_xor_sync(0xffffffffu, upper ? lo : hi, o));
    };
    float v = m[0];
    if constexpr (G == 2) v = merge(b0, m[0], m[1], 1);
    if constexpr (G == 4) v = merge(b1, merge(b0, m[0], m[1], 1), merge(b0, m[2], m[3], 1), 2);
#pragma unroll
    for (int o = 4 * G; o >= G; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The scales of a lane's groups and their reciprocals, rounded to nearest,
// from group_max's answer: each lane forms those of one group (a division and
// a reciprocal take some 30 instructions).
template <int FMT, int G>
__device__ __forceinline__ void tile_scales(float own, float (&s)[G], float (&r)[G]) {
    const int lane = threadIdx.x & 31;
    const float sc = fp8_block_scale<FMT>(own), rc = __frcp_rn(sc);
#pragma unroll
    for (int g = 0; g < G; g++) {
        s[g] = G == 1 ? sc : __shfl_sync(0xffffffffu, sc, (lane & ~(G - 1)) + g);
        r[g] = G == 1 ? rc : __shfl_sync(0xffffffffu, rc, (lane & ~(G - 1)) + g);
    }
}

// The absmax of a lane's values in each of its groups, without the NaNs, and
// whether any value of the warp is not finite (`odd`): a maximum that keeps
// NaN shows it, and only then the values are looked at again.
template <int G>
__device__ __forceinline__ void tile_absmax(const f2 (&v)[8], float (&m)[G], bool& odd) {
    constexpr int P = 8 / G;
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) {
        m[g] = 0.f;
#pragma unroll
        for (int i = 0; i < P; i++) {
            float a, b;
            split_f2(v[P * g + i], a, b);
            m[g] = absmax_nan(m[g], a, b);
        }
        top = G == 1 ? m[g] : absmax_nan(top, m[g], 0.f);
    }
    odd = __any_sync(0xffffffffu, !(top < __int_as_float(0x7f800000)));
    if (odd) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            m[g] = 0.f;
#pragma unroll
            for (int i = 0; i < P; i++) {
                float a, b;
                split_f2(v[P * g + i], a, b);
                m[g] = fmaxf(fmaxf(m[g], fabsf(a)), fabsf(b));  // fmaxf passes a NaN over
            }
        }
    }
}

// The codes of a lane's 16 values, 4 to a word in order, given the scale s of
// each of its groups and r = RN(1 / s).  Finite tiles: the quotients are at most max_finite and
// a rounding, which the converter brings back to max_finite, so nothing is
// clamped and no NaN is looked for; scales of at least 2^-60 take
// fp8_product.h's correction of x * RN(1 / s) (the correctly rounded
// quotient), smaller ones the division.
template <int FMT, int G>
__device__ __forceinline__ void tile_codes(const f2 (&v)[8], const float (&s)[G], const float (&rs)[G], bool odd,
                                           uint32_t (&w)[4]) {
    bool product = !odd;
#pragma unroll
    for (int g = 0; g < G; g++) product = product && s[g] >= 8.6736174e-19f;
    if (product) {
        // -x / s, so that a zero comes out with its sign: the residual of
        // x = -0 would be +0, and take the sign of the quotient with it
        f2 r[G], p[G];
#pragma unroll
        for (int g = 0; g < G; g++) r[g] = make_f2(-rs[g]), p[g] = make_f2(s[g]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int g = i * G / 4;
            uint32_t c[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f2 x = v[2 * i + h], y = mul_f2(x, r[g]);
                float q0, q1;
                split_f2(fma_f2(fma_f2(y, p[g], x), r[g], y), q0, q1);
                c[h] = FMT == RENG_FP8_E4M3 ? cvt_e4m3x2(q0, q1) : cvt_e5m2x2(q0, q1);
            }
            w[i] = __byte_perm(c[0], c[1], 0x5410) ^ 0x80808080u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float sc = s[i * G / 4];
            float a, b, c, d;
            split_f2(v[2 * i], a, b);
            split_f2(v[2 * i + 1], c, d);
            w[i] = encode2<FMT>(div_host(a, sc), div_host(b, sc)) | encode2<FMT>(div_host(c, sc), div_host(d, sc)) << 16;
        }
    }
}

// A lane's codes of group g into the row at column c (G 1, 2: of this lane).
template <int G>
__device__ __forceinline__ void tile_store_codes(uint8_t* row, int c, int cols, int g, const uint32_t (&w)[4]) {
    if (G == 1) {
        *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if (G == 2) {
        *reinterpret_cast<uint2*>(row + c) = make_uint2(w[(2 * g) & 3], w[(2 * g + 1) & 3]);
    } else {
        uint8_t* p = row + c + (threadIdx.x & 31);
        if (c + kFp8Group <= cols) {
#pragma unroll
            for (int i = 0; i < 4; i++) p[32 * i] = (uint8_t)(w[g] >> (8 * i));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (c + 32 * i + (int)(threadIdx.x & 31) < cols) p[32 * i] = (uint8_t)(w[g] >> (8 * i));
        }
    }
}

}  // namespace reng
