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
#include <type_traits>

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

// Sum over the CTA, the same bits on every thread (warps added in order).
// `red` alternates between two buffers, so one barrier is enough: a buffer is
// written again only after the barrier of the other's sum.
__device__ __forceinline__ float cta_sum(float v, float (&red)[2][32], int& turn) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    float* r = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) r[warp] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < nw; w++) s += r[w];
    return s;
}

__device__ __forceinline__ float inv_rms(float sum, float n, float eps) { return 1.0f / sqrtf(sum / n + eps); }

// The 4 groups of a warp tile of one row: the first column of the lane's
// values in each (VEC: in its own).
template <bool VEC>
struct Tile {
    static constexpr int G = VEC ? 1 : kTileGroups;
    int64_t c[G];
    bool live[G];
    __device__ __forceinline__ Tile(int64_t tile, int64_t cols) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int g = 0; g < G; g++) {
            c[g] = tile * (kTileGroups * kFp8Group) + (VEC ? lane * 16 : g * kFp8Group);
            live[g] = c[g] < cols;
        }
    }
};

template <bool KEEP, int TYPE, bool VEC>
__device__ __forceinline__ void tile_load(const void* base, int64_t at, const Tile<VEC>& t, int64_t cols,
                                          Raw16<TYPE, VEC>& r) {
    const char* row = static_cast<const char*>(base) + at * (TYPE == RENG_TYPE_BF16 ? 2 : 4);
    raw_zero(r);
    if constexpr (VEC) {
        if (t.live[0]) raw_load<TYPE, KEEP>(row + t.c[0] * (TYPE == RENG_TYPE_BF16 ? 2 : 4), r);
    } else {
#pragma unroll
        for (int g = 0; g < kTileGroups; g++)
            if (t.live[g]) raw_load<TYPE, KEEP>(row, t.c[g], cols, g, r);
    }
}

// The same as floats, of a type known at run time (uniform).
template <bool KEEP, bool VEC>
__device__ __forceinline__ void tile_floats(const void* base, int type, int64_t at, const Tile<VEC>& t, int64_t cols,
                                            float (&v)[16]) {
    if (type == RENG_TYPE_BF16) {
        Raw16<RENG_TYPE_BF16, VEC> r;
        tile_load<KEEP>(base, at, t, cols, r);
        raw_floats(r, v);
    } else {
        Raw16<RENG_TYPE_F32, VEC> r;
        tile_load<KEEP>(base, at, t, cols, r);
        raw_floats(r, v);
    }
}

template <int TYPE, bool VEC>
__device__ __forceinline__ void tile_store(void* base, int64_t at, const Tile<VEC>& t, int64_t cols,
                                           const float (&v)[16]) {
    if constexpr (VEC) {
        if (!t.live[0]) return;
        if (TYPE == RENG_TYPE_BF16) {
            uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at + t.c[0]);
#pragma unroll
            for (int i = 0; i < 2; i++)
                p[i] = make_uint4(bf16x2(v[8 * i], v[8 * i + 1]), bf16x2(v[8 * i + 2], v[8 * i + 3]),
                                  bf16x2(v[8 * i + 4], v[8 * i + 5]), bf16x2(v[8 * i + 6], v[8 * i + 7]));
        } else {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at + t.c[0]);
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
    } else {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int64_t c = t.c[e >> 2] + 32 * (e & 3) + lane;
            if (c < cols) {
                if (TYPE == RENG_TYPE_BF16)
                    static_cast<uint16_t*>(base)[at + c] = __bfloat16_as_ushort(__float2bfloat16_rn(v[e]));
                else static_cast<float*>(base)[at + c] = v[e];
            }
        }
    }
}

// u of a tile becomes the branch's share of y: normed, gained, gated; then
// y += scale * u, rounded to y's type.
template <int TR, bool VEC>
__device__ __forceinline__ void tile_residual(const NormArgs& a, int64_t row, const Tile<VEC>& t, float inv,
                                              float (&u)[16], float (&y)[16]) {
    float g[16];
    if (a.post) {
        tile_floats<true, VEC>(a.post, RENG_TYPE_F32, 0, t, a.cols, g);
#pragma unroll
        for (int i = 0; i < 16; i++) u[i] = u[i] * inv * g[i];
    }
    if (a.gate) {
        tile_floats<true, VEC>(a.gate, a.tg, row * a.ldg, t, a.cols, g);
#pragma unroll
        for (int i = 0; i < 16; i++) u[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < 16; i++) y[i] = fmaf(a.scale, u[i], y[i]);
    if (TR == RENG_TYPE_BF16) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint32_t p = bf16x2(y[i], y[i + 1]);
            y[i] = bf16lo(p), y[i + 1] = bf16hi(p);
        }
    }
}

template <int FMT, bool VEC>
__device__ __forceinline__ void tile_emit_fp8(const NormArgs& a, int64_t row, const Tile<VEC>& t,
                                              const float (&h)[16]) {
    constexpr int G = Tile<VEC>::G;
    const int lane = threadIdx.x & 31;
    uint32_t m[G];
    bool odd;
    tile_absmax<VEC>(h, m, odd);
    group_max<VEC>(m);
    float s[G];
#pragma unroll
    for (int g = 0; g < G; g++) s[g] = fp8_block_scale<FMT>(__uint_as_float(m[g]));
    const uint4 q = tile_codes<FMT, VEC>(h, s, odd);
    uint8_t* dst = static_cast<uint8_t*>(a.h) + row * a.ldh;
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (!t.live[g]) continue;
        if ((lane & (VEC ? 7 : 31)) == 0) a.scales[row * a.lds + t.c[g] / kFp8Group] = s[g];
        if constexpr (VEC) *reinterpret_cast<uint4*>(dst + t.c[g]) = q;
        else store_codes(dst, t.c[g], a.cols, g == 0 ? q.x : g == 1 ? q.y : g == 2 ? q.z : q.w);
    }
}

// h of a tile (whole warps: the FP8 groups shuffle).
template <bool VEC>
__device__ __forceinline__ void tile_emit(const NormArgs& a, int64_t row, const Tile<VEC>& t, float inv,
                                          const float (&y)[16]) {
    float h[16];
    if (a.pre) {
        tile_floats<true, VEC>(a.pre, RENG_TYPE_F32, 0, t, a.cols, h);
#pragma unroll
        for (int i = 0; i < 16; i++) h[i] = y[i] * inv * h[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) h[i] = y[i] * inv;
    }
    if (a.out == OUT_BF16) tile_store<RENG_TYPE_BF16, VEC>(a.h, row * a.ldh, t, a.cols, h);
    else if (a.out == OUT_F32) tile_store<RENG_TYPE_F32, VEC>(a.h, row * a.ldh, t, a.cols, h);
    else if (a.out == OUT_E4M3) tile_emit_fp8<RENG_FP8_E4M3, VEC>(a, row, t, h);
    else tile_emit_fp8<RENG_FP8_E5M2, VEC>(a, row, t, h);
}

__device__ __forceinline__ float square_sum(const float (&v)[16], float s) {
#pragma unroll
    for (int i = 0; i < 16; i++) s = fmaf(v[i], v[i], s);
    return s;
}

// One CTA per row, the row in registers: C warp tiles per warp.
template <int TB, int TR, bool VEC, int C>
__global__ void __launch_bounds__(512) k_block_norm(NormArgs a) {
    __shared__ float red[2][32];
    int turn = 0;
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const float n = (float)a.cols;
    pdl_wait();
    pdl_launch();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float y[C][16], u[C][16];
#pragma unroll
        for (int k = 0; k < C; k++) {
            const Tile<VEC> t(k * nw + warp, a.cols);
            Raw16<TR, VEC> r;
            Raw16<TB, VEC> b;
            tile_load<false>(a.residual, row * a.ldr, t, a.cols, r);
            if (a.branch) tile_load<false>(a.branch, row * a.ldb, t, a.cols, b);
            raw_floats(r, y[k]);
            if (a.branch) raw_floats(b, u[k]);
        }
        if (a.branch) {
            float inv = 1.f;
            if (a.post) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < C; k++) s = square_sum(u[k], s);
                inv = inv_rms(cta_sum(s, red, turn), n, a.eps);
            }
#pragma unroll
            for (int k = 0; k < C; k++) {
                const Tile<VEC> t(k * nw + warp, a.cols);
                tile_residual<TR, VEC>(a, row, t, inv, u[k], y[k]);
                tile_store<TR, VEC>(a.y, row * a.ldy, t, a.cols, y[k]);
            }
        }
        if (a.out == OUT_NONE) continue;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < C; k++) s = square_sum(y[k], s);
        const float inv = inv_rms(cta_sum(s, red, turn), n, a.eps);
#pragma unroll
        for (int k = 0; k < C; k++) tile_emit<VEC>(a, row, Tile<VEC>(k * nw + warp, a.cols), inv, y[k]);
    }
}

// Rows too long for the registers: three passes over the columns, each warp
// reading back only what it wrote itself.
template <int TB, int TR, bool VEC>
__global__ void __launch_bounds__(512) k_block_norm_long(NormArgs a) {
    __shared__ float red[2][32];
    int turn = 0;
    const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const float n = (float)a.cols;
    const int64_t tiles = (a.cols + kTileGroups * kFp8Group - 1) / (kTileGroups * kFp8Group);
    pdl_wait();
    pdl_launch();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float inv = 1.f;
        if (a.branch && a.post) {
            float s = 0.f;
            for (int64_t i = warp; i < tiles; i += nw) {
                float u[16];
                tile_floats<false, VEC>(a.branch, TB, row * a.ldb, Tile<VEC>(i, a.cols), a.cols, u);
                s = square_sum(u, s);
            }
            inv = inv_rms(cta_sum(s, red, turn), n, a.eps);
        }
        float s = 0.f;
        for (int64_t i = warp; i < tiles; i += nw) {
            const Tile<VEC> t(i, a.cols);
            float y[16];
            tile_floats<false, VEC>(a.residual, TR, row * a.ldr, t, a.cols, y);
            if (a.branch) {
                float u[16];
                tile_floats<false, VEC>(a.branch, TB, row * a.ldb, t, a.cols, u);
                tile_residual<TR, VEC>(a, row, t, inv, u, y);
                tile_store<TR, VEC>(a.y, row * a.ldy, t, a.cols, y);
            }
            s = square_sum(y, s);
        }
        if (a.out == OUT_NONE) continue;
        inv = inv_rms(cta_sum(s, red, turn), n, a.eps);
        for (int64_t i = warp; i < tiles; i += nw) {
            const Tile<VEC> t(i, a.cols);
            float y[16];
            if (a.branch) tile_floats<false, VEC>(a.y, TR, row * a.ldy, t, a.cols, y);
            else tile_floats<false, VEC>(a.residual, TR, row * a.ldr, t, a.cols, y);
            tile_emit<VEC>(a, row, t, inv, y);
        }
    }
}

template <int TB, int TR, bool VEC>
cudaError_t launch_row(const NormArgs& a, int sms, cudaStream_t st) {
    constexpr int kTile = kTileGroups * kFp8Group;
    const int64_t tiles = (a.cols + kTile - 1) / kTile;
    const dim3 grid((unsigned)std::min<int64_t>(a.rows, (int64_t)1 << 30));
    if (tiles <= 16) return launch_ops(k_block_norm<TB, TR, VEC, 1>, grid, dim3(32 * (unsigned)tiles), 0, st, a);
    if (tiles <= 32)
        return launch_ops(k_block_norm<TB, TR, VEC, 2>, grid, dim3(32 * (unsigned)((tiles + 1) / 2)), 0, st, a);
    return launch_ops(k_block_norm_long<TB, TR, VEC>, grid, dim3(512), 0, st, a);
}

int launch(const NormArgs& a, bool vec, cudaStream_t st) {
    int sms = 0;
    RENG_CUDA_TRY(current_sms(&sms));
    constexpr int B = RENG_TYPE_BF16, F = RENG_TYPE_F32;
    auto pick = [&](auto v) {
        constexpr bool V = decltype(v)::value;
        if (a.tr == B) return a.tb == B ? launch_row<B, B, V>(a, sms, st) : launch_row<F, B, V>(a, sms, st);
        return a.tb == B ? launch_row<B, F, V>(a, sms, st) : launch_row<F, F, V>(a, sms, st);
    };
    const cudaError_t e = vec ? pick(std::true_type()) : pick(std::false_type());
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
    a.tb = d->branch ? d->branch_type : d->residual_type;
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
    const bool vec = a.cols % 16 == 0 && aligned(a.branch, a.ldb, eb, 16) && aligned(a.residual, a.ldr, er, 16) &&
                     aligned(a.gate, a.ldg, eg, 16) && aligned(y, a.ldy, er, 16) &&
                     aligned(h, a.ldh, eh, 16) && aligned(a.post, 0, 4, 16) && aligned(a.pre, 0, 4, 16);
    return launch(a, vec, (cudaStream_t)stream);
}
