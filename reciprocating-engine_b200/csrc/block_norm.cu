// The step between two blocks of a decoder, one pass over each row:
//
//   u = branch                       the block's output
//   u = u * r(u) * post_gain         (optional) a norm after the block
//   u = u * gate                     (optional) per element or per column
//   y = round(residual + scale * u)  the residual stream, rounded once to its type
//   h = y * r(y) * pre_gain          the next block's input, from y as stored
//
// with r(v) = 1 / sqrt(mean(v^2) + eps) over the row, sums and norms in f32,
// and h written in bf16, in f32 or as FP8 codes with one scale per 1 x 128
// group (the operand of the block-scaled product): the FP8 form rounds h
// once, from f32.  Replaces, for an 8-bit path, the reference's residual add
// and RMSNorm nodes (crates/reng-synapse/src/model.rs:738-742).
#include <algorithm>
#include <cmath>
#include <string>

#include "fp8_encode.cuh"
#include "ops.cuh"

namespace reng {
namespace {

enum Out : int { OUT_NONE = 0, OUT_BF16, OUT_F32, OUT_E4M3, OUT_E5M2 };

struct NormArgs {
    const void *branch, *residual, *gate;
    void *y, *h;
    float* scales;
    const float *post, *pre;
    int64_t rows, cols, ldb, ldr, ldg, ldy, ldh, lds;
    int tb, tr, tg;  // element types (RENG_TYPE_*); y has tr
    int out;
    float scale, eps;
};

__device__ __forceinline__ int esize(int type) { return type == RENG_TYPE_BF16 ? 2 : 4; }

// 8 values of a row whose type is known at run time (the branch is uniform).
// Plain loads: y may be written over residual.
template <bool VEC>
__device__ __forceinline__ void load8t(const void* base, int type, int64_t elem, int64_t c, int64_t cols,
                                       float (&v)[8]) {
    if (VEC) {
        if (type == RENG_TYPE_BF16) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem + c);
            v[0] = bf16lo(u.x), v[1] = bf16hi(u.x), v[2] = bf16lo(u.y), v[3] = bf16hi(u.y);
            v[4] = bf16lo(u.z), v[5] = bf16hi(u.z), v[6] = bf16lo(u.w), v[7] = bf16hi(u.w);
        } else {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elem + c);
            const float4 a = p[0], b = p[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = 0.f;
        if (c + i < cols)
            v[i] = type == RENG_TYPE_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(base)[elem + c + i])
                                          : static_cast<const float*>(base)[elem + c + i];
    }
}

template <bool VEC>
__device__ __forceinline__ void store8t(void* base, int type, int64_t elem, int64_t c, int64_t cols,
                                        const float (&v)[8]) {
    if (VEC) {
        if (type == RENG_TYPE_BF16) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + elem + c) =
                make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                           pack_bf16x2(v[6], v[7]));
        } else {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + elem + c);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (c + i < cols) {
            if (type == RENG_TYPE_BF16)
                static_cast<uint16_t*>(base)[elem + c + i] = f32_to_bf16_bits(v[i]);
            else
                static_cast<float*>(base)[elem + c + i] = v[i];
        }
}

// Sum over the CTA, the same bits on every thread (warps added in order).
__device__ __forceinline__ float cta_sum(float v, float* red) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < nw; w++) s += red[w];
    __syncthreads();
    return s;
}

__device__ __forceinline__ float inv_rms(float sum, float n, float eps) { return 1.0f / sqrtf(sum / n + eps); }

// h of 8 columns; every lane of the warp calls it (the FP8 groups shuffle).
template <bool VEC>
__device__ __forceinline__ void emit(const NormArgs& a, int64_t row, int64_t c, bool live, float inv,
                                     const float (&y)[8]) {
    float h[8];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = 0.f;
    if (live) {
        if (a.pre) {
            load8t<VEC>(a.pre, RENG_TYPE_F32, 0, c, a.cols, h);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = c + i < a.cols ? y[i] * inv * h[i] : 0.f;
    }
    if (a.out == OUT_BF16 || a.out == OUT_F32) {
        if (live) store8t<VEC>(a.h, a.out == OUT_BF16 ? RENG_TYPE_BF16 : RENG_TYPE_F32, row * a.ldh, c, a.cols, h);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) m = fp8_absmax(m, h[i]);
    m = half_warp_max(m);
    if (!live) return;
    uint8_t* codes = static_cast<uint8_t*>(a.h) + row * a.ldh;
    float s;
    uint2 q;
    if (a.out == OUT_E4M3) {
        s = fp8_block_scale<RENG_FP8_E4M3>(m);
        q = fp8_encode8<RENG_FP8_E4M3>(h, s, m);
    } else {
        s = fp8_block_scale<RENG_FP8_E5M2>(m);
        q = fp8_encode8<RENG_FP8_E5M2>(h, s, m);
    }
    if ((c & (kFp8Group - 1)) == 0) a.scales[row * a.lds + c / kFp8Group] = s;
    store_codes8<VEC>(codes, c, a.cols, q);
}

// y of 8 columns from the branch values u (already normed and gained).
template <bool VEC>
__device__ __forceinline__ void residual8(const NormArgs& a, int64_t row, int64_t c, float (&u)[8], float (&y)[8]) {
    if (a.gate) {
        float g[8];
        load8t<VEC>(a.gate, a.tg, row * a.ldg, c, a.cols, g);
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        y[i] = fmaf(a.scale, u[i], y[i]);
        if (a.tr == RENG_TYPE_BF16) y[i] = round_bf16(y[i]);
    }
}

// One CTA per row, the row in registers: C chunks of 8 columns per thread.
template <int C>
__global__ void __launch_bounds__(1024) k_block_norm(NormArgs a) {
    __shared__ float red[32];
    pdl_wait();
    pdl_launch();
    const int T = blockDim.x;
    const float n = (float)a.cols;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float y[C][8], u[C][8];
#pragma unroll
        for (int k = 0; k < C; k++) {
            const int64_t c = ((int64_t)k * T + threadIdx.x) * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) y[k][i] = 0.f, u[k][i] = 0.f;
            if (c < a.cols) {
                load8t<true>(a.residual, a.tr, row * a.ldr, c, a.cols, y[k]);
                if (a.branch) load8t<true>(a.branch, a.tb, row * a.ldb, c, a.cols, u[k]);
            }
        }
        if (a.branch) {
            if (a.post) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < C; k++)
#pragma unroll
                    for (int i = 0; i < 8; i++) s = fmaf(u[k][i], u[k][i], s);
                const float inv = inv_rms(cta_sum(s, red), n, a.eps);
#pragma unroll
                for (int k = 0; k < C; k++) {
                    const int64_t c = ((int64_t)k * T + threadIdx.x) * 8;
                    if (c < a.cols) {
                        float g[8];
                        load8t<true>(a.post, RENG_TYPE_F32, 0, c, a.cols, g);
#pragma unroll
                        for (int i = 0; i < 8; i++) u[k][i] = u[k][i] * inv * g[i];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < C; k++) {
                const int64_t c = ((int64_t)k * T + threadIdx.x) * 8;
                if (c < a.cols) {
                    residual8<true>(a, row, c, u[k], y[k]);
                    store8t<true>(a.y, a.tr, row * a.ldy, c, a.cols, y[k]);
                }
            }
        }
        if (a.out == OUT_NONE) continue;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < C; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) s = fmaf(y[k][i], y[k][i], s);
        const float inv = inv_rms(cta_sum(s, red), n, a.eps);
#pragma unroll
        for (int k = 0; k < C; k++) {
            const int64_t c = ((int64_t)k * T + threadIdx.x) * 8;
            emit<true>(a, row, c, c < a.cols, inv, y[k]);
        }
    }
}

// Any width, pitch and alignment: the row in three passes over its columns
// (each thread reads back only what it wrote itself).
__global__ void __launch_bounds__(1024) k_block_norm_any(NormArgs a) {
    __shared__ float red[32];
    pdl_wait();
    pdl_launch();
    const float n = (float)a.cols;
    const int64_t stride = (int64_t)blockDim.x * 8;
    const int64_t end = (a.cols + 127) / 128 * 128;  // whole groups: a group's lanes stay together
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float inv = 1.f;
        if (a.branch && a.post) {
            float s = 0.f;
            for (int64_t c = threadIdx.x * 8; c < a.cols; c += stride) {
                float u[8];
                load8t<false>(a.branch, a.tb, row * a.ldb, c, a.cols, u);
#pragma unroll
                for (int i = 0; i < 8; i++) s = fmaf(u[i], u[i], s);
            }
            inv = inv_rms(cta_sum(s, red), n, a.eps);
        }
        const void* src = a.branch ? a.y : a.residual;
        const int64_t lds = a.branch ? a.ldy : a.ldr;
        float s = 0.f;
        for (int64_t c = threadIdx.x * 8; c < a.cols; c += stride) {
            float y[8];
            load8t<false>(a.residual, a.tr, row * a.ldr, c, a.cols, y);
            if (a.branch) {
                float u[8];
                load8t<false>(a.branch, a.tb, row * a.ldb, c, a.cols, u);
                if (a.post) {
                    float g[8];
                    load8t<false>(a.post, RENG_TYPE_F32, 0, c, a.cols, g);
#pragma unroll
                    for (int i = 0; i < 8; i++) u[i] = u[i] * inv * g[i];
                }
                residual8<false>(a, row, c, u, y);
                store8t<false>(a.y, a.tr, row * a.ldy, c, a.cols, y);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) s = fmaf(y[i], y[i], s);
        }
        if (a.out == OUT_NONE) continue;
        inv = inv_rms(cta_sum(s, red), n, a.eps);
        for (int64_t c0 = 0; c0 < end; c0 += stride) {
            const int64_t c = c0 + threadIdx.x * 8;
            float y[8];
            load8t<false>(src, a.tr, row * lds, c, a.cols, y);
            emit<false>(a, row, c, c < a.cols, inv, y);
        }
    }
}

int launch(const NormArgs& a, bool vec, cudaStream_t st) {
    int sms = 0;
    RENG_CUDA_TRY(current_sms(&sms));
    const int64_t chunks = a.cols / 8;
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, (int64_t)1 << 20);
    auto threads = [](int64_t n) { return (unsigned)((n + 31) / 32 * 32); };
    cudaError_t e;
    if (!vec || chunks > 4096) {
        const unsigned t = std::min<unsigned>(1024u, threads((a.cols + 7) / 8));
        e = launch_ops(k_block_norm_any, dim3(grid), dim3(t), 0, st, a);
    } else if (chunks <= 1024) {
        e = launch_ops(k_block_norm<1>, dim3(grid), dim3(threads(chunks)), 0, st, a);
    } else if (chunks <= 2048) {
        e = launch_ops(k_block_norm<2>, dim3(grid), dim3(threads((chunks + 1) / 2)), 0, st, a);
    } else {
        e = launch_ops(k_block_norm<4>, dim3(grid), dim3(threads((chunks + 3) / 4)), 0, st, a);
    }
    if (e != cudaSuccess) return fail(RENG_E_CUDA, std::string("reng_block_norm: ") + cudaGetErrorString(e));
    return RENG_OK;
}

bool type_ok(int t) { return t == RENG_TYPE_BF16 || t == RENG_TYPE_F32; }
int host_esize(int t) { return t == RENG_TYPE_BF16 ? 2 : 4; }

}  // namespace
}  // namespace reng

using namespace reng;

extern "C" int reng_block_norm(const reng_block_norm_desc *d, void *stream) {
    const std::string f = "reng_block_norm: ";
    RENG_CHECK_ARG(d != nullptr, f + "desc is NULL");
    RENG_CHECK_ARG(d->rows >= 0 && d->cols >= 1, f + "rows >= 0 and cols >= 1, not " + std::to_string(d->rows) +
                                                     " x " + std::to_string(d->cols));
    RENG_CHECK_ARG(type_ok(d->residual_type) && (!d->branch || type_ok(d->branch_type)) &&
                       (!d->gate || type_ok(d->gate_type)),
                   f + "unknown element type");
    RENG_CHECK_ARG(d->out >= RENG_NORM_NONE && d->out <= RENG_NORM_E5M2, f + "unknown output kind");
    RENG_CHECK_ARG(std::isfinite(d->eps) && d->eps >= 0.f && std::isfinite(d->scale), f + "eps / scale not finite, or eps below 0");
    const bool fp8 = d->out == RENG_NORM_E4M3 || d->out == RENG_NORM_E5M2;
    RENG_CHECK_ARG(d->branch || d->out != RENG_NORM_NONE, f + "no branch and no output: nothing to do");
    RENG_CHECK_ARG(d->branch || (!d->gate && !d->post_gain), f + "a gate or a post norm without a branch");
    RENG_CHECK_ARG(ops_pitch_ok(d->rows, d->cols, d->ld_residual) &&
                       (!d->branch || (ops_pitch_ok(d->rows, d->cols, d->ld_branch) &&
                                       ops_pitch_ok(d->rows, d->cols, d->ld_y))) &&
                       (!d->gate || d->ld_gate == 0 || ops_pitch_ok(d->rows, d->cols, d->ld_gate)) &&
                       (d->out == RENG_NORM_NONE || ops_pitch_ok(d->rows, d->cols, d->ld_h)) &&
                       (!fp8 || ops_pitch_ok(d->rows, ops_groups(d->cols), d->ld_scales)),
                   f + "a row pitch below its row, or sizes above 2^40 elements");
    if (d->rows == 0) return RENG_OK;
    RENG_CHECK_ARG(d->residual && (!d->branch || d->y) && (d->out == RENG_NORM_NONE || d->h) && (!fp8 || d->h_scales),
                   f + "NULL buffer");
    NormArgs a{};
    a.branch = d->branch;
    a.residual = d->residual;
    a.gate = d->gate;
    a.y = d->y;
    a.h = d->h;
    a.scales = d->h_scales;
    a.post = d->post_gain;
    a.pre = d->pre_gain;
    a.rows = d->rows;
    a.cols = d->cols;
    a.ldb = d->ld_branch;
    a.ldr = d->ld_residual;
    a.ldg = d->ld_gate;
    a.ldy = d->ld_y;
    a.ldh = d->ld_h;
    a.lds = d->ld_scales;
    a.tb = d->branch_type;
    a.tr = d->residual_type;
    a.tg = d->gate_type;
    a.out = d->out;
    a.scale = d->scale;
    a.eps = d->eps;
    auto aligned = [](const void* p, int64_t ld, int esz, int n) { return !p || ops_aligned(p, ld * esz, n); };
    const int eb = host_esize(a.tb), er = host_esize(a.tr), eg = host_esize(a.tg);
    const int eh = fp8 ? 1 : (a.out == OUT_BF16 ? 2 : 4);
    const void* y = d->branch ? d->y : nullptr;
    const void* h = a.out == OUT_NONE ? nullptr : d->h;
    RENG_CHECK_ARG(aligned(a.branch, a.ldb, eb, eb) && aligned(a.residual, a.ldr, er, er) &&
                       aligned(a.gate, a.ldg, eg, eg) && aligned(y, a.ldy, er, er) && aligned(h, a.ldh, eh, eh) &&
                       aligned(a.post, 0, 4, 4) && aligned(a.pre, 0, 4, 4) &&
                       (!fp8 || aligned(a.scales, a.lds, 4, 4)),
                   f + "a buffer is not aligned to its element");
    const bool vec = a.cols % 8 == 0 && aligned(a.branch, a.ldb, eb, 16) && aligned(a.residual, a.ldr, er, 16) &&
                     aligned(a.gate, a.ldg, eg, 16) && aligned(y, a.ldy, er, 16) &&
                     aligned(h, a.ldh, eh, fp8 ? 8 : 16) && aligned(a.post, 0, 4, 16) && aligned(a.pre, 0, 4, 16);
    return launch(a, vec, (cudaStream_t)stream);
}
