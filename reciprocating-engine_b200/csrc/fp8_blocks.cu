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
    int64_t groups;  // ceil(cols / 128)
};

// g / (1 + exp(-g)) * u: expf overflows to infinity for g below about -88,
// where the quotient is the (negative) zero that the limit is.
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// 1 x 128 groups: a half-warp owns one group, each lane 8 consecutive values,
// so a group's absmax is a 4-step shuffle and the codes leave from registers.
template <int TYPE, int FMT, bool VEC, bool SWIGLU>
__global__ void __launch_bounds__(256) k_fp8_groups(GroupArgs a) {
    constexpr int esz = TYPE == RENG_TYPE_BF16 ? 2 : 4;
    pdl_wait();
    pdl_launch();
    const int sub = threadIdx.x & 15;
    const int64_t total = a.rows * a.groups;
    const int64_t step = (int64_t)gridDim.x * 16;
    const int64_t first = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    // the two groups of a warp may end at different counts: the loop runs to
    // the warp's last one, so the shuffles always have all 32 lanes
    const int64_t warp_first = first & ~(int64_t)1;
    for (int64_t w = warp_first; w < total; w += step) {
        const int64_t t = w + (first & 1);
        const bool live = t < total;
        const int64_t row = live ? t / a.groups : 0, grp = live ? t - row * a.groups : 0;
        const int64_t c = grp * kFp8Group + sub * 8;
        float v[8];
        float m = 0.f;
        if (live) {
            load8<TYPE, VEC>(static_cast<const char*>(a.x) + (size_t)row * a.ldx * esz, c, a.cols, v);
            if (SWIGLU) {
                float u[8];
                load8<TYPE, VEC>(static_cast<const char*>(a.up) + (size_t)row * a.ldx * esz, c, a.cols, u);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = swiglu(v[i], u[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) m = fp8_absmax(m, v[i]);
        }
        m = half_warp_max(m);
        if (live) {
            const float s = fp8_block_scale<FMT>(m);
            if (sub == 0) a.scales[row * a.lds + grp] = s;
            store_codes8<VEC>(a.codes + row * a.ldc, c, a.cols, fp8_encode8<FMT>(v, s, m));
        }
    }
}

// 128 x 128 blocks: one CTA per block, the block in registers between the
// absmax and the codes (16 lanes across a row's 128 columns, 8 rows each).
template <int TYPE, int FMT, bool VEC>
__global__ void __launch_bounds__(256) k_fp8_blocks(GroupArgs a) {
    constexpr int esz = TYPE == RENG_TYPE_BF16 ? 2 : 4;
    __shared__ float red[8];
    pdl_wait();
    pdl_launch();
    const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4, warp = threadIdx.x >> 5;
    const int64_t total = (a.rows + kFp8Group - 1) / kFp8Group * a.groups;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t rb = b / a.groups, grp = b - rb * a.groups;
        const int64_t c = grp * kFp8Group + sub * 8;
        float v[8][8];
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t row = rb * kFp8Group + r0 + 16 * i;
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = 0.f;
            if (row < a.rows)
                load8<TYPE, VEC>(static_cast<const char*>(a.x) + (size_t)row * a.ldx * esz, c, a.cols, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) m = fp8_absmax(m, v[i][e]);
        m = warp_max(m);
        if ((threadIdx.x & 31) == 0) red[warp] = m;
        __syncthreads();
        m = red[0];
#pragma unroll
        for (int w = 1; w < 8; w++) m = fmaxf(m, red[w]);
        __syncthreads();  // red is rewritten by the next block
        const float s = fp8_block_scale<FMT>(m);
        if (threadIdx.x == 0) a.scales[rb * a.lds + grp] = s;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t row = rb * kFp8Group + r0 + 16 * i;
            if (row < a.rows) store_codes8<VEC>(a.codes + row * a.ldc, c, a.cols, fp8_encode8<FMT>(v[i], s, m));
        }
    }
}

template <int TYPE, int FMT, bool VEC>
cudaError_t launch_blocks(const GroupArgs& a, int block_rows, bool swiglu, cudaStream_t st) {
    int sms = 0;
    cudaError_t e = current_sms(&sms);
    if (e != cudaSuccess) return e;
    if (block_rows > 1) {
        const int64_t total = (a.rows + kFp8Group - 1) / kFp8Group * a.groups;
        return launch_ops(k_fp8_blocks<TYPE, FMT, VEC>, dim3((unsigned)std::min<int64_t>(total, 1 << 20)), dim3(256),
                          0, st, a);
    }
    const int64_t total = a.rows * a.groups;
    const unsigned grid = (unsigned)std::min<int64_t>((total + 15) / 16, (int64_t)sms * 8);
    return swiglu ? launch_ops(k_fp8_groups<TYPE, FMT, VEC, true>, dim3(grid), dim3(256), 0, st, a)
                  : launch_ops(k_fp8_groups<TYPE, FMT, VEC, false>, dim3(grid), dim3(256), 0, st, a);
}

template <int TYPE, int FMT>
cudaError_t pick_vec(const GroupArgs& a, int block_rows, bool swiglu, cudaStream_t st) {
    const int esz = TYPE == RENG_TYPE_BF16 ? 2 : 4;
    const bool vec = ops_aligned(a.x, a.ldx * esz, 16) && (!swiglu || ops_aligned(a.up, a.ldx * esz, 16)) &&
                     ops_aligned(a.codes, a.ldc, 8);
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
    GroupArgs a{x, nullptr, rows, cols, ldx, codes, ldc, scales, lds, ops_groups(cols)};
    return quantize("reng_fp8_quantize_blocks", a, type, block_rows, fmt, false, (cudaStream_t)stream);
}

extern "C" int reng_fp8_swiglu_quantize(const void *gate, const void *up, int type, int64_t rows, int64_t cols,
                                        int64_t ldx, int fmt, uint8_t *codes, int64_t ldc, float *scales, int64_t lds,
                                        void *stream) {
    const int rc =
        check_quantize("reng_fp8_swiglu_quantize: ", gate, up, type, rows, cols, ldx, fmt, codes, ldc, scales, lds);
    if (rc || rows == 0) return rc;
    GroupArgs a{gate, up, rows, cols, ldx, codes, ldc, scales, lds, ops_groups(cols)};
    return quantize("reng_fp8_swiglu_quantize", a, type, 1, fmt, true, (cudaStream_t)stream);
}
