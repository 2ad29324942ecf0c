// The block quantizers: FP8 codes with one f32 scale per 1 x 128 group of a
// row (activations) or per 128 x 128 block (weights), the operands of the
// block-scaled product (gemm_fp8.cu).
//
//   a = max |x| over the block (NaN never taken), s = a / max_finite (1 if
//   a = 0), code = encode(x / s): the arithmetic of the per-row quantizer
//   (fp8_quant.cu, after crates/reng-fp8/src/lib.rs:519-563) on a block.
//
// and the same of h = silu(g) * u, the input of a decoder's down projection,
// so the activation never goes through HBM at 16 bits.
#include <algorithm>
#include <string>
#include <type_traits>

#include "ops.cuh"
#include "fp8_encode.cuh"

namespace reng {
namespace {

struct GroupArgs {
    const void* x;   // values; the gate of the SwiGLU form
    const void* up;  // SwiGLU only
    int64_t rows, ldx;
    int cols;
    uint8_t* codes;
    int64_t ldc;
    float* scales;
    int64_t lds;
    uint32_t blocks;  // groups, or 128 x 128 blocks
    FastDiv per_row;  // of one row (of blocks)
};

// exp(-g), or exp(g) 2^208 (FAR), by the hardware's ex2: 2^t with t = g log2(e)
// in two parts, so that the rounding of t (which |g| magnifies) does not reach
// the result: 2^(hi + lo) = 2^hi (1 + lo ln 2).
template <bool FAR>
__device__ __forceinline__ f2 exp_f2(f2 g) {
    constexpr float s = FAR ? 1.f : -1.f;
    const f2 hi = mul_f2(g, make_f2(s * 1.44269504f)), neg = mul_f2(hi, make_f2(-1.0f));
    const f2 lo =
        fma_f2(g, make_f2(s * 1.33497580e-8f), mul_f2(fma_f2(g, make_f2(s * 1.44269504f), neg), make_f2(0.693147181f)));
    float e0, e1;
    split_f2(FAR ? add_f2(hi, make_f2(208.f)) : hi, e0, e1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(e0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(e1));
    const f2 e = make_f2(e0, e1);
    return fma_f2(e, lo, e);
}

// silu(g) u where exp(-|g|) is nothing beside 1: g u, or g exp(g) u, which a
// large u brings back into the f32 range though exp(g) has left it.  exp(g) is
// taken 2^208 too large (the shift of hi is exact, and exp(-200) 2^208 still
// normal; under -200 every product is below f32's smallest), half of that given
// back by u first, so that nothing overflows, or loses bits that count, on the
// way.  -inf, which has no limit, gives NaN.
__device__ __forceinline__ f2 swiglu_far(f2 g, f2 u) {
    float g0, g1, p0, p1, r0, r1;
    split_f2(g, g0, g1);
    const f2 w = mul_f2(g, exp_f2<true>(make_f2(fmaxf(g0, -300.f), fmaxf(g1, -300.f)))), half = make_f2(4.93038066e-32f);  // 2^-104
    split_f2(mul_f2(g, u), p0, p1);
    split_f2(mul_f2(mul_f2(mul_f2(u, half), w), half), r0, r1);
    return make_f2(g0 < 0.f ? r0 : p0, g1 < 0.f ? r1 : p1);
}

// v[i] = silu(v[i]) u[i].  The quotient is rcp's, corrected by its residual.
// About 6 roundings in all.  Where 1 + exp(-g) nears the end of the f32 range
// (g from -86.5 down, and infinities and NaN), a pair that some lane has
// there is formed again by swiglu_far; activations have such gates in single
// columns (a test for each pair, then: SwiGLU of 8192 x 14336 bf16 with a gate
// of 87 in a quarter of its warp tiles 119 us, all pairs again 127, and 114
// with the far products taken as zeros).
__device__ __forceinline__ void swiglu(f2 (&v)[8], const f2 (&u)[8]) {
    float top = 0.f;
    f2 h[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const f2 g = v[i], d = add_f2(exp_f2<false>(g), make_f2(1.0f));
        float d0, d1;
        split_f2(d, d0, d1);
        top = absmax_nan(top, d0, d1);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d0) : "f"(d0));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d1) : "f"(d1));
        const f2 r = make_f2(d0, d1), y = mul_f2(g, r), ny = mul_f2(y, make_f2(-1.0f));
        h[i] = mul_f2(fma_f2(fma_f2(ny, d, g), r, y), u[i]);
    }
    if (__any_sync(0xffffffffu, !(top < 3.6e37f))) {  // under exp(86.5): a value's form does not depend on its neighbours'
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float g0, g1, f0, f1, h0, h1;
            split_f2(v[i], g0, g1);
            const bool far0 = !(g0 > -86.5f && g0 < 1e30f), far1 = !(g1 > -86.5f && g1 < 1e30f);
            if (!__any_sync(0xffffffffu, far0 || far1)) continue;
            split_f2(swiglu_far(v[i], u[i]), f0, f1);
            split_f2(h[i], h0, h1);
            h[i] = make_f2(far0 ? f0 : h0, far1 ? f1 : h1);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = h[i];
}

template <int TYPE>
__device__ __forceinline__ const void* elem(const void* base, int64_t at) {
    return static_cast<const char*>(base) + at * (TYPE == RENG_TYPE_BF16 ? 2 : 4);
}

// The scales and codes of a warp tile's values (SWIGLU: of silu(x) u).
template <int TYPE, int FMT, int G, bool SWIGLU>
__device__ __forceinline__ void encode_tile(const Raw16<TYPE, G>& x, const Raw16<TYPE, G>& u, float (&s)[G], uint32_t (&w)[4]) {
    f2 v[8];
    raw_floats(x, v);
    if (SWIGLU) {
        f2 f[8];
        raw_floats(u, f);
        swiglu(v, f);
    }
    float m[G], r[G];
    bool odd;
    tile_absmax(v, m, odd);
    tile_scales<FMT>(group_max(m), s, r);
    tile_codes<FMT>(v, s, r, odd, w);
}

// 1 x 128 groups: one warp tile of 4 consecutive groups (of any rows) each,
// codes and scales straight from registers.  4 CTAs an SM: with the loads'
// latency and the exponentials 3 leave issue slots free, and 5 spill (SwiGLU of
// 8192 x 14336 bf16 on 3, 4 and 5: 122, 117 and 132 us,
// without the far form).
template <int TYPE, int FMT, int G, bool SWIGLU>
__global__ void __launch_bounds__(256, 4) k_fp8_groups(GroupArgs a) {
    const uint32_t t0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kTileGroups;
    pdl_wait();
    pdl_launch();
    Raw16<TYPE, G> x, u;
    float s[G];
    uint32_t w[4];
    if constexpr (G == 4) {
        // by elements, 4 whole groups of one row (most tiles): one base address
        // and no test (SwiGLU of 4346 x 9669 bf16: 10 us of 74)
        const uint32_t row = a.per_row.div(t0), grp = t0 - row * a.per_row.d;
        if (t0 < a.blocks && grp + kTileGroups <= (uint32_t)a.cols / kFp8Group) {
            const int c = (int)(grp * kFp8Group);
            const void* from = elem<TYPE>(a.x, row * a.ldx + c);
#pragma unroll
            for (int g = 0; g < G; g++) raw_load<TYPE, false, true>(from, g * kFp8Group, 0, g, x);
            if (SWIGLU) {
                const void* up = elem<TYPE>(a.up, row * a.ldx + c);
#pragma unroll
                for (int g = 0; g < G; g++) raw_load<TYPE, false, true>(up, g * kFp8Group, 0, g, u);
            }
            encode_tile<TYPE, FMT, G, SWIGLU>(x, u, s, w);
            uint8_t* to = a.codes + (row * a.ldc + c);
            float* scales = a.scales + (row * a.lds + grp);
#pragma unroll
            for (int g = 0; g < G; g++) {
                if (lane_first<G>()) scales[g] = s[g];
                tile_store_codes<G>(to, g * kFp8Group, G * kFp8Group, g, w);
            }
            return;
        }
    }
    uint32_t row[G], grp[G];
    int c[G];
    bool live[G];
    raw_zero(x);
    if (SWIGLU) raw_zero(u);
#pragma unroll
    for (int g = 0; g < G; g++) {
        const uint32_t t = t0 + lane_group<G>(g);
        row[g] = a.per_row.div(t);
        grp[g] = t - row[g] * a.per_row.d;
        c[g] = (int)(grp[g] * kFp8Group) + lane_col<G>();
        live[g] = t < a.blocks && c[g] < a.cols;
        if (!live[g]) continue;
        const int64_t at = row[g] * a.ldx;
        if constexpr (G < 4) {
            raw_load<TYPE>(elem<TYPE>(a.x, at + c[g]), g, x);
            if (SWIGLU) raw_load<TYPE>(elem<TYPE>(a.up, at + c[g]), g, u);
        } else {
            raw_load<TYPE>(elem<TYPE>(a.x, at), c[g], a.cols, g, x);
            if (SWIGLU) raw_load<TYPE>(elem<TYPE>(a.up, at), c[g], a.cols, g, u);
        }
    }
    encode_tile<TYPE, FMT, G, SWIGLU>(x, u, s, w);
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (!live[g]) continue;
        if (lane_first<G>()) a.scales[row[g] * a.lds + grp[g]] = s[g];
        tile_store_codes<G>(a.codes + row[g] * a.ldc, c[g], a.cols, g, w);
    }
}

// 128 x 128 blocks: one CTA per block, the block in registers between the
// absmax and the codes: 4 tiles per warp, a tile 4 rows of the block.  3 CTAs
// an SM by elements and of f32, 4 of bf16 pieces (6061 x 6962 bf16 by elements:
// 46, 39 and 41 us with 2, 3 and 4; 4096 x 14336 in pieces 31.2 and 28.4 with
// 3 and 4).
template <int TYPE, int FMT, int G>
__global__ void __launch_bounds__(256, G == 4 || TYPE == RENG_TYPE_F32 ? 3 : 4) k_fp8_blocks(GroupArgs a) {
    __shared__ float red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rb = a.per_row.div(blockIdx.x), grp = blockIdx.x - rb * a.per_row.d;
    const int c = (int)(grp * kFp8Group) + lane_col<G>();
    // the row of this lane's group g in tile i
    auto row_of = [&](int i, int g) { return (int64_t)rb * kFp8Group + 32 * i + 4 * warp + lane_group<G>(g); };
    pdl_wait();
    pdl_launch();
    Raw16<TYPE, G> x[4];
    auto load = [&](auto all) {
        constexpr bool kAll = decltype(all)::value;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!kAll) raw_zero(x[i]);
#pragma unroll
            for (int g = 0; g < G; g++) {
                const int64_t row = row_of(i, g);
                if (!kAll && (row >= a.rows || c >= a.cols)) continue;
                if constexpr (G < 4) raw_load<TYPE>(elem<TYPE>(a.x, row * a.ldx + c), g, x[i]);
                else raw_load<TYPE, false, kAll>(elem<TYPE>(a.x, row * a.ldx), c, a.cols, g, x[i]);
            }
        }
    };
    if ((int64_t)(rb + 1) * kFp8Group <= a.rows && (int)(grp + 1) * kFp8Group <= a.cols) load(std::true_type());
    else load(std::false_type());
    float top = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f2 v[8];
        float m[G];
        bool o;
        raw_floats(x[i], v);
        tile_absmax(v, m, o);
        odd = odd || o;
#pragma unroll
        for (int g = 0; g < G; g++) top = fmaxf(top, m[g]);
    }
    top = warp_max(top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = fmaxf(top, red[w]);
    // a warp whose values are finite still divides by an infinite scale
    odd = odd || top == __int_as_float(0x7f800000);
    // the codes start from the raw values again: as floats they would take
    // twice the registers meanwhile, and the SM hold one CTA less
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int k = 0; k < Raw16<TYPE, G>::N; k++) asm volatile("" : "+r"(x[i].w[k]));
    float s[G], r[G];
    s[0] = fp8_block_scale<FMT>(top);
    r[0] = __frcp_rn(s[0]);
#pragma unroll
    for (int g = 1; g < G; g++) s[g] = s[0], r[g] = r[0];
    if (threadIdx.x == 0) a.scales[rb * a.lds + grp] = s[0];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f2 v[8];
        raw_floats(x[i], v);
        uint32_t w[4];
        tile_codes<FMT>(v, s, r, odd, w);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int64_t row = row_of(i, g);
            if (row < a.rows && c < a.cols) tile_store_codes<G>(a.codes + row * a.ldc, c, a.cols, g, w);
        }
    }
}

template <int TYPE, int FMT, int G>
cudaError_t launch_blocks(const GroupArgs& a, int block_rows, bool swiglu, cudaStream_t st) {
    if (block_rows > 1) return launch_ops(k_fp8_blocks<TYPE, FMT, G>, dim3(a.blocks), dim3(256), 0, st, a);
    const dim3 grid((a.blocks + 31) / 32);  // 8 warps of 4 groups
    return swiglu ? launch_ops(k_fp8_groups<TYPE, FMT, G, true>, grid, dim3(256), 0, st, a)
                  : launch_ops(k_fp8_groups<TYPE, FMT, G, false>, grid, dim3(256), 0, st, a);
}

template <int TYPE, int FMT>
cudaError_t pick_vec(const GroupArgs& a, int block_rows, bool swiglu, cudaStream_t st) {
    const int esz = TYPE == RENG_TYPE_BF16 ? 2 : 4;
    // whole 16-column pieces on 16 bytes, whole 8-column pieces, or any row
    // (333 x 5000 f32: 2.7 us in pieces of 8, 3.7 by elements)
    const bool rows = ops_aligned(a.x, a.ldx * esz, 16) && (!swiglu || ops_aligned(a.up, a.ldx * esz, 16));
    if (rows && a.cols % 16 == 0 && ops_aligned(a.codes, a.ldc, 16)) return launch_blocks<TYPE, FMT, 1>(a, block_rows, swiglu, st);
    if (rows && a.cols % 8 == 0 && ops_aligned(a.codes, a.ldc, 8)) return launch_blocks<TYPE, FMT, 2>(a, block_rows, swiglu, st);
    return launch_blocks<TYPE, FMT, 4>(a, block_rows, swiglu, st);
}

int quantize(const char* who, const GroupArgs& a, int type, int block_rows, int fmt, bool swiglu, cudaStream_t st) {
    cudaError_t e;
    if (type == RENG_TYPE_BF16)
        e = fmt == RENG_FP8_E4M3 ? pick_vec<RENG_TYPE_BF16, RENG_FP8_E4M3>(a, block_rows, swiglu, st)
                                 : pick_vec<RENG_TYPE_BF16, RENG_FP8_E5M2>(a, block_rows, swiglu, st);
    else
        e = fmt == RENG_FP8_E4M3 ? pick_vec<RENG_TYPE_F32, RENG_FP8_E4M3>(a, block_rows, swiglu, st)
                                 : pick_vec<RENG_TYPE_F32, RENG_FP8_E5M2>(a, block_rows, swiglu, st);
    if (e != cudaSuccess) return fail(RENG_E_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
    return RENG_OK;
}

int check_quantize(const std::string& f, const void* x, const void* up, int type, int64_t rows, int64_t cols,
                   int64_t ldx, int fmt, const void* codes, int64_t ldc, const void* scales, int64_t lds) {
    RENG_CHECK_ARG(rows >= 0 && cols >= 1 && cols <= kOpsMaxCols, f + "rows >= 0 and cols in [1, 2^30], not " + std::to_string(rows) + " x " +
                                               std::to_string(cols));
    RENG_CHECK_ARG(type == RENG_TYPE_BF16 || type == RENG_TYPE_F32, f + "unknown element type");
    RENG_CHECK_ARG(fmt == RENG_FP8_E4M3 || fmt == RENG_FP8_E5M2, f + "unknown format");
    const int64_t groups = ops_groups(cols);
    RENG_CHECK_ARG(ops_pitch_ok(rows, cols, ldx) && ops_pitch_ok(rows, cols, ldc) && ops_pitch_ok(rows, groups, lds),
                   f + "a row pitch below its row, or sizes above 2^40 elements");
    // one index per group: codes alone would be 2^38 bytes beyond this
    RENG_CHECK_ARG(groups <= INT32_MAX && rows <= INT32_MAX / groups, f + "more than 2^31 groups");
    if (rows == 0) return RENG_OK;
    RENG_CHECK_ARG(x && up && codes && scales, f + "NULL buffer");
    const uintptr_t esz = type == RENG_TYPE_BF16 ? 2 : 4;
    RENG_CHECK_ARG((uintptr_t)x % esz == 0 && (uintptr_t)up % esz == 0 && (uintptr_t)scales % 4 == 0,
                   f + "a buffer is not aligned to its element");
    return RENG_OK;
}

}  // namespace
}  // namespace reng

using namespace reng;

extern "C" int reng_fp8_quantize_blocks(const void *x, int type, int64_t rows, int64_t cols, int64_t ldx,
                                        int block_rows, int fmt, uint8_t *codes, int64_t ldc, float *scales,
                                        int64_t lds, void *stream) {
    RENG_CHECK_ARG(block_rows == 1 || block_rows == kFp8Group, "reng_fp8_quantize_blocks: block_rows must be 1 or 128");
    const int rc = check_quantize("reng_fp8_quantize_blocks: ", x, x, type, rows, cols, ldx, fmt, codes, ldc, scales, lds);
    if (rc || rows == 0) return rc;
    const int64_t groups = ops_groups(cols), per = (rows + block_rows - 1) / block_rows * groups;
    GroupArgs a{x, nullptr, rows, ldx, (int)cols, codes, ldc, scales, lds, (uint32_t)per, FastDiv((uint32_t)groups)};
    return quantize("reng_fp8_quantize_blocks", a, type, block_rows, fmt, false, (cudaStream_t)stream);
}

extern "C" int reng_fp8_swiglu_quantize(const void *gate, const void *up, int type, int64_t rows, int64_t cols,
                                        int64_t ldx, int fmt, uint8_t *codes, int64_t ldc, float *scales, int64_t lds,
                                        void *stream) {
    const int rc =
        check_quantize("reng_fp8_swiglu_quantize: ", gate, up, type, rows, cols, ldx, fmt, codes, ldc, scales, lds);
    if (rc || rows == 0) return rc;
    const int64_t groups = ops_groups(cols);
    GroupArgs a{gate, up, rows, ldx, (int)cols, codes, ldc, scales, lds, (uint32_t)(rows * groups), FastDiv((uint32_t)groups)};
    return quantize("reng_fp8_swiglu_quantize", a, type, 1, fmt, true, (cudaStream_t)stream);
}
