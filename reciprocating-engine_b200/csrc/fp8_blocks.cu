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

#include "ops.cuh"
#include "fp8_encode.cuh"

namespace reng {
namespace {

struct GroupArgs {
    const void* x;   // values; the gate of the SwiGLU form
    const void* up;  // SwiGLU only
    int64_t rows, cols, ldx;
    uint8_t* codes;
    int64_t ldc;
    float* scales;
    int64_t lds;
    uint32_t blocks;  // groups, or 128 x 128 blocks
    FastDiv per_row;  // of one row (of blocks)
};

// g / (1 + exp(-g)) * u.  exp(-g) is 2^t by the hardware's ex2, t = -g log2(e)
// in two parts so that the rounding of t (which |g| magnifies) does not reach
// the result: 2^(hi + lo) = 2^hi (1 + lo ln 2).  It overflows to infinity for
// g below about -88, where the quotient is the (negative) zero of the limit;
// where 2^t is out of reach of the sum the correction is left out.
// About 10 roundings in all (ex2 4, rcp 2, the rest one each).
__device__ __forceinline__ float swiglu(float g, float u) {
    const float hi = __fmul_rn(g, -1.44269504f);
    const float lo = fmaf(g, -1.92596299e-8f, fmaf(g, -1.44269504f, -hi));
    float e, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(hi));
    e = fabsf(hi) < 126.f ? fmaf(e, lo * 0.693147181f, e) : e;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * r * u;
}

template <int TYPE, bool VEC>
__device__ __forceinline__ const void* elem(const void* base, int64_t at) {
    return static_cast<const char*>(base) + at * (TYPE == RENG_TYPE_BF16 ? 2 : 4);
}

// 1 x 128 groups: one warp tile of 4 consecutive groups (of any rows) each,
// codes and scales straight from registers.
template <int TYPE, int FMT, bool VEC, bool SWIGLU>
__global__ void __launch_bounds__(256) k_fp8_groups(GroupArgs a) {
    constexpr int G = VEC ? 1 : kTileGroups;
    const int lane = threadIdx.x & 31;
    const uint32_t t0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kTileGroups + (VEC ? lane >> 3 : 0);
    pdl_wait();
    pdl_launch();
    uint32_t row[G], grp[G];
    int64_t c[G];
    bool live[G];
    Raw16<TYPE, VEC> x, u;
    raw_zero(x);
    if (SWIGLU) raw_zero(u);
#pragma unroll
    for (int g = 0; g < G; g++) {
        row[g] = a.per_row.div(t0 + g);
        grp[g] = t0 + g - row[g] * a.per_row.d;
        c[g] = (int64_t)grp[g] * kFp8Group + (VEC ? (lane & 7) * 16 : 0);
        live[g] = t0 + g < a.blocks && c[g] < a.cols;
        if (live[g]) {
            const int64_t at = row[g] * a.ldx;
            if constexpr (VEC) {
                raw_load<TYPE>(elem<TYPE, VEC>(a.x, at + c[g]), x);
                if (SWIGLU) raw_load<TYPE>(elem<TYPE, VEC>(a.up, at + c[g]), u);
            } else {
                raw_load<TYPE>(elem<TYPE, VEC>(a.x, at), c[g], a.cols, g, x);
                if (SWIGLU) raw_load<TYPE>(elem<TYPE, VEC>(a.up, at), c[g], a.cols, g, u);
            }
        }
    }
    float v[16];
    raw_floats(x, v);
    if (SWIGLU) {
        float w[16];
        raw_floats(u, w);
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = swiglu(v[i], w[i]);
    }
    uint32_t m[G];
    bool odd;
    tile_absmax<VEC>(v, m, odd);
    group_max<VEC>(m);
    float s[G];
#pragma unroll
    for (int g = 0; g < G; g++) s[g] = fp8_block_scale<FMT>(__uint_as_float(m[g]));
    const uint4 q = tile_codes<FMT, VEC>(v, s, odd);
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (!live[g]) continue;
        if ((lane & (VEC ? 7 : 31)) == 0) a.scales[row[g] * a.lds + grp[g]] = s[g];
        uint8_t* dst = a.codes + row[g] * a.ldc;
        if constexpr (VEC) *reinterpret_cast<uint4*>(dst + c[g]) = q;
        else store_codes(dst, c[g], a.cols, g == 0 ? q.x : g == 1 ? q.y : g == 2 ? q.z : q.w);
    }
}

// 128 x 128 blocks: one CTA per block, the block in registers between the
// absmax and the codes: 4 tiles per warp, a tile 4 rows of the block.
template <int TYPE, int FMT, bool VEC>
__global__ void __launch_bounds__(256) k_fp8_blocks(GroupArgs a) {
    constexpr int G = VEC ? 1 : kTileGroups;
    __shared__ uint32_t red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rb = a.per_row.div(blockIdx.x), grp = blockIdx.x - rb * a.per_row.d;
    const int64_t c = (int64_t)grp * kFp8Group + (VEC ? (lane & 7) * 16 : 0);
    // the first row of tile i (VEC: this lane's row)
    auto row_of = [&](int i) { return (int64_t)rb * kFp8Group + 32 * i + 4 * warp + (VEC ? lane >> 3 : 0); };
    pdl_wait();
    pdl_launch();
    Raw16<TYPE, VEC> x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        raw_zero(x[i]);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int64_t row = row_of(i) + g;
            if (row < a.rows && c < a.cols) {
                if constexpr (VEC) raw_load<TYPE>(elem<TYPE, VEC>(a.x, row * a.ldx + c), x[i]);
                else raw_load<TYPE>(elem<TYPE, VEC>(a.x, row * a.ldx), c, a.cols, g, x[i]);
            }
        }
    }
    uint32_t top = 0u;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float v[16];
        uint32_t m[G];
        bool o;
        raw_floats(x[i], v);
        tile_absmax<VEC>(v, m, o);
        odd = odd || o;
#pragma unroll
        for (int g = 0; g < G; g++) top = max(top, m[g]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = max(top, red[w]);
    // a warp whose values are finite still divides by an infinite scale
    odd = odd || top >= 0x7f800000u;
    float s[G];
#pragma unroll
    for (int g = 0; g < G; g++) s[g] = fp8_block_scale<FMT>(__uint_as_float(top));
    if (threadIdx.x == 0) a.scales[rb * a.lds + grp] = s[0];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float v[16];
        raw_floats(x[i], v);
        const uint4 q = tile_codes<FMT, VEC>(v, s, odd);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int64_t row = row_of(i) + g;
            if (row >= a.rows || c >= a.cols) continue;
            uint8_t* dst = a.codes + row * a.ldc;
            if constexpr (VEC) *reinterpret_cast<uint4*>(dst + c) = q;
            else store_codes(dst, c, a.cols, g == 0 ? q.x : g == 1 ? q.y : g == 2 ? q.z : q.w);
        }
    }
}

template <int TYPE, int FMT, bool VEC>
cudaError_t launch_blocks(const GroupArgs& a, int block_rows, bool swiglu, cudaStream_t st) {
    if (block_rows > 1) return launch_ops(k_fp8_blocks<TYPE, FMT, VEC>, dim3(a.blocks), dim3(256), 0, st, a);
    const dim3 grid((a.blocks + 31) / 32);  // 8 warps of 4 groups
    return swiglu ? launch_ops(k_fp8_groups<TYPE, FMT, VEC, true>, grid, dim3(256), 0, st, a)
                  : launch_ops(k_fp8_groups<TYPE, FMT, VEC, false>, grid, dim3(256), 0, st, a);
}

template <int TYPE, int FMT>
cudaError_t pick_vec(const GroupArgs& a, int block_rows, bool swiglu, cudaStream_t st) {
    const int esz = TYPE == RENG_TYPE_BF16 ? 2 : 4;
    const bool vec = a.cols % 16 == 0 && ops_aligned(a.x, a.ldx * esz, 16) &&
                     (!swiglu || ops_aligned(a.up, a.ldx * esz, 16)) && ops_aligned(a.codes, a.ldc, 16);
    return vec ? launch_blocks<TYPE, FMT, true>(a, block_rows, swiglu, st)
               : launch_blocks<TYPE, FMT, false>(a, block_rows, swiglu, st);
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
    RENG_CHECK_ARG(rows >= 0 && cols >= 1, f + "rows >= 0 and cols >= 1, not " + std::to_string(rows) + " x " +
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
    GroupArgs a{x, nullptr, rows, cols, ldx, codes, ldc, scales, lds, (uint32_t)per, FastDiv((uint32_t)groups)};
    return quantize("reng_fp8_quantize_blocks", a, type, block_rows, fmt, false, (cudaStream_t)stream);
}

extern "C" int reng_fp8_swiglu_quantize(const void *gate, const void *up, int type, int64_t rows, int64_t cols,
                                        int64_t ldx, int fmt, uint8_t *codes, int64_t ldc, float *scales, int64_t lds,
                                        void *stream) {
    const int rc =
        check_quantize("reng_fp8_swiglu_quantize: ", gate, up, type, rows, cols, ldx, fmt, codes, ldc, scales, lds);
    if (rc || rows == 0) return rc;
    const int64_t groups = ops_groups(cols);
    GroupArgs a{gate, up, rows, cols, ldx, codes, ldc, scales, lds, (uint32_t)(rows * groups), FastDiv((uint32_t)groups)};
    return quantize("reng_fp8_swiglu_quantize", a, type, 1, fmt, true, (cudaStream_t)stream);
}
