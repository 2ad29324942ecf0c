// The block-scaled FP8 product (gemm_fp8.cu) for the few token rows of a
// decode step, where every weight byte is read once and only that counts.
//
// mma.sync m16n8k32 on the codes as they lie: 16 weight rows are the MMA's M,
// up to 8 (or twice 8) token rows its N.  A block's 128 products are summed
// by four MMAs from zero, and the sum is scaled into f32 accumulators (4 per
// lane and 8 tokens).  Within a block the order of k does not matter, so lane
// (g, q) takes 16 consecutive bytes of row g at 16 q and hands them to the
// MMAs as the k its fragments name; the token rows are read the same way.
// That makes every load 16 bytes wide with no staging, no barrier and no TMEM
// round trip per block (which costs the tcgen05 form some 470 cycles a block,
// whatever its width).
// One CTA owns 16 weight rows; its warps split K and add their partials in
// warp order through shared memory, so the result is deterministic.  8 warps
// with three blocks (6 KB) each in flight, two CTAs an SM (one above 8 token
// rows); or 4 warps with four blocks, three (two) CTAs, where those hold all
// CTAs of a launch at once and the former do not (us, 8 and 4 warps: 1 row
// 6144 x 4096 8.1 / 6.9, 5120 x 5120 9.0 / 7.9, but 4096 x 4096 5.4 / 6.2, 8192
// x 4096 9.6 / 10.8; 16 rows 4096 x 4096 8.8 / 7.9, but 5120 x 5120 13.6 / 14.5).
#include <algorithm>
#include <string>

#include "fp8_encode.cuh"
#include "ops.cuh"

namespace reng {
namespace {

constexpr int kTile = 16;   // weight rows of a CTA
// K splits of a CTA (its warps: 8 or 4), a warp's blocks in flight, CTAs of an SM
constexpr int ahead(int warps) { return warps == 8 ? 3 : 4; }
constexpr int ctas(int warps, int mt) { return (warps == 8 ? 2 : 3) - (mt == 1 ? 0 : 1); }

struct Gemv8Args {
    const uint8_t *x, *w;
    const float *sx, *sw;
    void* y;
    int64_t ldx, ldw, ldsx, ldsw, ldy;
    int M, N, K, kb;
    int y_f32;
};

template <int XF, int WF>
__device__ __forceinline__ void mma_f8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
#define RENG_MMA(W, X)                                                                                     \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32." W "." X ".f32 {%0, %1, %2, %3}, "                \
                 "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                                           \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                          \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if (WF == RENG_FP8_E4M3 && XF == RENG_FP8_E4M3) RENG_MMA("e4m3", "e4m3");
    else if (WF == RENG_FP8_E4M3) RENG_MMA("e4m3", "e5m2");
    else if (XF == RENG_FP8_E4M3) RENG_MMA("e5m2", "e4m3");
    else RENG_MMA("e5m2", "e5m2");
#undef RENG_MMA
}

// The last n < 16 codes of a row (out of line: it is taken at most once a row).
__device__ __noinline__ void tail16(const uint8_t* p, int n, uint32_t (&w)[4]) {
    for (int i = 0; i < n; i++) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
}

// 16 codes of a row from column k on; those at or past K are zeros, and
// nothing past the row's K codes is read.
// RAGGED: K is no multiple of 16.
template <bool STREAM, bool RAGGED>
__device__ __forceinline__ uint4 codes16(const uint8_t* row, int k, int K) {
    if (RAGGED ? k + 16 <= K : k < K) return STREAM ? ldg_stream(row + k) : *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (RAGGED && k < K) tail16(row + k, K - k, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// What one lane holds of a block: rows g and g + 8 of the weights and row g
// of each 8 tokens, 16 codes at 16 q of both 64-byte halves, and the scales
// of its two output columns.
template <int MT>
struct Block {
    uint4 w[2][2], x[MT][2];
    float sw, sx[MT][2];
};

template <int MT, int XF, int WF, bool RAGGED, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, ctas(kWarps, MT)) k_gemv_fp8(const Gemv8Args a) {
    constexpr int kAhead = ahead(kWarps);
    __shared__ float red[kWarps][MT * 8][kTile + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int n0 = blockIdx.x * kTile;
    const int b0 = (int)((long long)warp * a.kb / kWarps), b1 = (int)((long long)(warp + 1) * a.kb / kWarps);
    const uint8_t* w0 = a.w + (size_t)min(n0 + g, a.N - 1) * a.ldw;      // rows past the matrix repeat its last:
    const uint8_t* w1 = a.w + (size_t)min(n0 + g + 8, a.N - 1) * a.ldw;  // their sums are not written
    const float* sw = a.sw + (size_t)(n0 / kFp8Group) * a.ldsw;
    pdl_wait();
    pdl_launch();
    auto load = [&](int b, Block<MT>& f) {
        const int k = b * kFp8Group + 16 * q;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f.w[0][h] = codes16<true, RAGGED>(w0, k + 64 * h, a.K);
            f.w[1][h] = codes16<true, RAGGED>(w1, k + 64 * h, a.K);
        }
        f.sw = sw[b];
#pragma unroll
        for (int t = 0; t < MT; t++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
                f.x[t][h] = 8 * t + g < a.M ? codes16<false, RAGGED>(a.x + (size_t)(8 * t + g) * a.ldx, k + 64 * h, a.K)
                                            : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int m = 8 * t + 2 * q + c;
                f.sx[t][c] = m < a.M ? a.sx[(size_t)m * a.ldsx + b] : 0.f;
            }
        }
    };
    float acc[MT][4];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[t][i] = 0.f;
    auto add = [&](const Block<MT>& f) {
#pragma unroll
        for (int t = 0; t < MT; t++) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                mma_f8<XF, WF>(d, f.w[0][h].x, f.w[1][h].x, f.w[0][h].y, f.w[1][h].y, f.x[t][h].x, f.x[t][h].y);
                mma_f8<XF, WF>(d, f.w[0][h].z, f.w[1][h].z, f.w[0][h].w, f.w[1][h].w, f.x[t][h].z, f.x[t][h].w);
            }
            const float s0 = f.sx[t][0] * f.sw, s1 = f.sx[t][1] * f.sw;
            acc[t][0] = fmaf(s0, d[0], acc[t][0]);
            acc[t][1] = fmaf(s1, d[1], acc[t][1]);
            acc[t][2] = fmaf(s0, d[2], acc[t][2]);
            acc[t][3] = fmaf(s1, d[3], acc[t][3]);
        }
    };
    Block<MT> f[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
        if (b0 + i < b1) load(b0 + i, f[i]);
    for (int b = b0; b < b1; b += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (b + i >= b1) break;
            add(f[i]);
            if (b + i + kAhead < b1) load(b + i + kAhead, f[i]);
        }
    }
    // lane (g, q) holds rows g, g + 8 of tokens 2 q, 2 q + 1
#pragma unroll
    for (int t = 0; t < MT; t++) {
        red[warp][8 * t + 2 * q][g] = acc[t][0];
        red[warp][8 * t + 2 * q + 1][g] = acc[t][1];
        red[warp][8 * t + 2 * q][g + 8] = acc[t][2];
        red[warp][8 * t + 2 * q + 1][g + 8] = acc[t][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 8 * kTile; i += 32 * kWarps) {
        const int m = i / kTile, n = n0 + i % kTile;
        if (m >= a.M || n >= a.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) v += red[w][m][i % kTile];
        const size_t at = (size_t)m * a.ldy + n;
        if (a.y_f32) static_cast<float*>(a.y)[at] = v;
        else static_cast<uint16_t*>(a.y)[at] = (uint16_t)bf16x2(v, 0.f);
    }
}

template <int MT, bool RAGGED, int W>
cudaError_t launch_warps(const Gemv8Args& a, unsigned tiles, int x_fmt, int w_fmt, cudaStream_t st) {
    const dim3 grid(tiles), block(32 * W);
    constexpr int E4 = RENG_FP8_E4M3, E5 = RENG_FP8_E5M2;
    if (w_fmt == E4)
        return x_fmt == E4 ? launch_ops(k_gemv_fp8<MT, E4, E4, RAGGED, W>, grid, block, 0, st, a)
                           : launch_ops(k_gemv_fp8<MT, E5, E4, RAGGED, W>, grid, block, 0, st, a);
    return x_fmt == E4 ? launch_ops(k_gemv_fp8<MT, E4, E5, RAGGED, W>, grid, block, 0, st, a)
                       : launch_ops(k_gemv_fp8<MT, E5, E5, RAGGED, W>, grid, block, 0, st, a);
}

template <int MT, bool RAGGED>
cudaError_t launch(const Gemv8Args& a, int x_fmt, int w_fmt, cudaStream_t st) {
    int sms = 0;
    const cudaError_t e = current_sms(&sms);
    if (e != cudaSuccess) return e;
    const int tiles = (a.N + kTile - 1) / kTile;
    return tiles > ctas(8, MT) * sms && tiles <= ctas(4, MT) * sms
               ? launch_warps<MT, RAGGED, 4>(a, (unsigned)tiles, x_fmt, w_fmt, st)
               : launch_warps<MT, RAGGED, 8>(a, (unsigned)tiles, x_fmt, w_fmt, st);
}

}  // namespace

int gemv_fp8_blocks(const uint8_t* x, int64_t ldx, const float* sx, int64_t ldsx, int x_fmt, const uint8_t* w,
                    int64_t ldw, const float* sw, int64_t ldsw, int w_fmt, int M, int N, int K, void* y, int y_type,
                    int64_t ldy, cudaStream_t st) {
    Gemv8Args a{x, w, sx, sw, y, ldx, ldw, ldsx, ldsw, ldy, M, N, K, (K + kFp8Group - 1) / kFp8Group, y_type == RENG_TYPE_F32};
    const bool ragged = K % 16 != 0;
    const cudaError_t e = M <= 8 ? (ragged ? launch<1, true>(a, x_fmt, w_fmt, st) : launch<1, false>(a, x_fmt, w_fmt, st))
                                 : (ragged ? launch<2, true>(a, x_fmt, w_fmt, st) : launch<2, false>(a, x_fmt, w_fmt, st));
    if (e != cudaSuccess) return fail(RENG_E_CUDA, std::string("reng_gemm_fp8_blocks: ") + cudaGetErrorString(e));
    return RENG_OK;
}

}  // namespace reng
