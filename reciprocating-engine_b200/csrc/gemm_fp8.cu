// The block-scaled FP8 product on the fifth-generation tensor cores:
//
//   y[m][n] = sum_b sx[m][b] * sw[n / 128][b] * sum_{k in block b} x[m][k] w[n][k]
//
// with x codes [M][K] carrying one f32 scale per 1 x 128 group and w codes
// [N][K] one per 128 x 128 block (the block quantizers' operands), y in bf16
// or f32.  The inner sums run on tcgen05.mma kind::f8f6f4 (8-bit operands as
// they lie in memory, f32 accumulation in TMEM over one 128-wide block); the
// scales, which change with every block, are applied when a block's sum is
// taken out of TMEM and added to f32 accumulators in registers:
//
//   acc[m][n] = fma(s, d[m][n], acc[m][n]),  s = sx[m][b] * sw[n / 128][b]
//
// Tile: 128 token rows (the MMA's M, one TMEM lane each) x BN weight rows
// (its N).  A lane's scale is one value for a whole 128-column weight block,
// so the step out of TMEM is one FMA per element.  Both operands are copied
// by TMA as {128 k, rows} boxes with the 128-byte swizzle, which is the
// K-major operand layout; rows and columns past the matrix read as zeros.
// Roles: warp 0 copies, warp 1 owns TMEM and issues the MMAs, warps 2.. hold
// the accumulators (a warp reads the TMEM lanes of its quarter, warp % 4).
// The MMAs of block b + 1 run into another TMEM buffer while block b's sum is
// added.  Few tiles (decode): K is split over the CTAs of a cluster, each
// leaves its f32 partial in its own shared memory and all of them add a share
// of the columns in rank order over distributed shared memory, so the result
// does not depend on arrival order and no workspace is needed.
// Every wait is bounded (tc.cuh); one that runs out records RENG_E_TIMEOUT in
// a device word, and the call's results are invalid.
#include <cooperative_groups.h>
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "fp8_encode.cuh"
#include "ops.cuh"
#include "tc.cuh"

namespace reng {
using namespace tc;

namespace {

constexpr int kRows = 128;       // token rows of a tile (the MMA's M)
constexpr int kBK = 128;         // k of a block: one swizzled row of 8-bit codes
constexpr int kMaxStages = 12;
constexpr int kMaxSplit = 8;     // a portable cluster

__device__ int g_fp8_gemm_err;   // set by a product whose waits ran out

struct Fp8Gemm {
    const float *sx, *sw;
    void* y;
    int64_t ldsx, ldsw, ldy;
    int M, N, kb;      // rows, columns, 128-k blocks
    int mt, nt;        // tiles
    int ks;            // K splits (CTAs of a cluster)
    int stages, mbox;  // pipeline stages, token rows of an x copy
    int y_f32, vec;    // output type; 16-byte stores allowed
    uint32_t idesc;
    int* err;
};

// 32 TMEM columns of this warp's lanes; the values are defined by tmem_wait32.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// The wait names the registers, so no use of them moves above it.
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void umma_f8(uint32_t tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::
            "r"(tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// A bounded wait whose outcome every lane of the warp shares.
__device__ __forceinline__ bool warp_wait(uint32_t b, uint32_t parity) {
    return __all_sync(0xffffffffu, bar_wait(b, parity));
}

// BN: weight rows of a tile; EW: accumulator warps (4, or 8 sharing the
// columns of a lane quarter); NB: TMEM buffers of BN columns.
template <int BN, int EW, int NB>
__global__ void __launch_bounds__(64 + 32 * EW, 1)
    k_gemm_fp8(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, Fp8Gemm a) {
    namespace cg = cooperative_groups;
    constexpr int CW = BN / (EW / 4);  // columns of one accumulator warp
    static_assert(CW % 32 == 0 && CW <= 128 && NB * BN <= 512, "tile shape");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) unsigned long long full[kMaxStages], empty[kMaxStages], tfull[NB], tempty[NB], drain;
    __shared__ uint32_t tmem_base_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem0 = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
    const uint32_t abytes = (uint32_t)a.mbox * kBK, bbytes = (uint32_t)BN * kBK;
    // x stages first: the MMA reads 128 rows from each, past a shorter box
    // into what follows, and the lanes of those rows are never used
    const uint32_t sA = smem0, sB = smem0 + (uint32_t)a.stages * abytes;
    auto bar = [](unsigned long long* b) { return (uint32_t)__cvta_generic_to_shared(b); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; s++) {
            bar_init(bar(&full[s]), 1);
            bar_init(bar(&empty[s]), 1);
        }
        for (int s = 0; s < NB; s++) {
            bar_init(bar(&tfull[s]), 1);
            bar_init(bar(&tempty[s]), EW);
        }
        bar_init(bar(&drain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&tmem_base_s);
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(NB * BN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base_s;
    pdl_wait();
    pdl_launch();

    const int rank = a.ks > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int k0 = (int)((long long)rank * a.kb / a.ks), k1 = (int)((long long)(rank + 1) * a.kb / a.ks);
    const long long tiles = (long long)a.mt * a.nt, tstep = gridDim.x / a.ks;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (long long t = blockIdx.x / a.ks; t < tiles && ok; t += tstep) {
                const int m0 = (int)(t % a.mt) * kRows, n0 = (int)(t / a.mt) * BN;
                for (int b = k0; b < k1; b++) {
                    if (issued >= a.stages && !(ok = bar_wait(bar(&empty[s]), ph ^ 1u))) break;
                    bar_expect_tx(bar(&full[s]), abytes + bbytes);
                    tensor_g2s(sA + (uint32_t)s * abytes, &xmap, b * kBK, m0, bar(&full[s]));
                    tensor_g2s(sB + (uint32_t)s * bbytes, &wmap, b * kBK, n0, bar(&full[s]));
                    issued = issued < a.stages ? issued + 1 : issued;
                    if (++s == a.stages) s = 0, ph ^= 1u;
                }
            }
            if (!ok) {
                atomicExch(a.err ? a.err : &g_fp8_gemm_err, RENG_E_TIMEOUT);
                // the last copy into each stage lands before the CTA may exit
                for (int i = 0; i < issued; i++) {
                    s = s == 0 ? (ph ^= 1u, a.stages - 1) : s - 1;
                    if (!bar_wait(bar(&full[s]), ph)) break;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int s = 0, d = 0, used = 0;
            uint32_t ph = 0, dph = 0;
            bool ok = true;
            for (long long t = blockIdx.x / a.ks; t < tiles && ok; t += tstep) {
                for (int b = k0; b < k1; b++) {
                    ok = bar_wait(bar(&full[s]), ph) && (used < NB || bar_wait(bar(&tempty[d]), dph ^ 1u));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
                        umma_f8(tmem + d * BN, umma_desc(sA + (uint32_t)s * abytes + kk * 32),
                                umma_desc(sB + (uint32_t)s * bbytes + kk * 32), a.idesc, kk ? 1u : 0u);
                    umma_commit(bar(&empty[s]));
                    umma_commit(bar(&tfull[d]));
                    used = used < NB ? used + 1 : used;
                    if (++s == a.stages) s = 0, ph ^= 1u;
                    if (++d == NB) d = 0, dph ^= 1u;
                }
            }
            if (!ok) atomicExch(a.err ? a.err : &g_fp8_gemm_err, RENG_E_TIMEOUT);
            // every MMA issued has completed before TMEM is freed
            umma_commit(bar(&drain));
            if (!bar_wait(bar(&drain), 0)) atomicExch(a.err ? a.err : &g_fp8_gemm_err, RENG_E_TIMEOUT);
        }
    } else {
        const int half = (warp - 2) >> 2;
        const int r = 32 * (warp & 3) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        int d = 0;
        uint32_t dph = 0;
        bool ok = true;
        for (long long t = blockIdx.x / a.ks; t < tiles; t += tstep) {
            const int m = (int)(t % a.mt) * kRows + r, n0 = (int)(t / a.mt) * BN + half * CW;
            const bool live = m < a.M;
            const bool any = m - lane < a.M && n0 < a.N;  // the warp has outputs in this tile
            float acc[CW];
#pragma unroll
            for (int c = 0; c < CW; c++) acc[c] = 0.f;
            const float* sx = a.sx + (size_t)(live ? m : 0) * a.ldsx;
            const float* sw = a.sw + (size_t)(n0 < a.N ? n0 / kBK : 0) * a.ldsw;
            float sn = any ? sx[k0] * sw[k0] : 0.f;
            for (int b = k0; b < k1; b++) {
                const float s = sn;
                if (any && b + 1 < k1) sn = sx[b + 1] * sw[b + 1];
                ok = ok && warp_wait(bar(&tfull[d]), dph);
                if (ok && any) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int g = 0; g < CW / 32; g++) {
                        uint32_t v[32];
                        tmem_ld32(tmem + lanes + d * BN + half * CW + g * 32, v);
                        tmem_wait32(v);
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            acc[g * 32 + e] = fmaf(s, __uint_as_float(v[e]), acc[g * 32 + e]);
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) bar_arrive(bar(&tempty[d]));
                if (++d == NB) d = 0, dph ^= 1u;
            }
            if (!ok) {
                if (lane == 0) atomicExch(a.err ? a.err : &g_fp8_gemm_err, RENG_E_TIMEOUT);
#pragma unroll
                for (int c = 0; c < CW; c++) acc[c] = __int_as_float(0x7fc00000);
            }
            if (a.ks > 1) {
                // partial[column][row], 129 rows apart: conflict-free both ways
                float* part = reinterpret_cast<float*>(smem_raw + (smem0 - (uint32_t)__cvta_generic_to_shared(smem_raw)));
                if (any)
#pragma unroll
                    for (int c = 0; c < CW; c++) part[(half * CW + c) * 129 + r] = acc[c];
            } else if (live && any) {
                if (a.y_f32) {
                    float* dst = static_cast<float*>(a.y) + (size_t)m * a.ldy + n0;
                    if (a.vec && n0 + CW <= a.N) {
#pragma unroll
                        for (int c = 0; c < CW; c += 4)
                            *reinterpret_cast<float4*>(dst + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
                    } else {
#pragma unroll
                        for (int c = 0; c < CW; c++)
                            if (n0 + c < a.N) dst[c] = acc[c];
                    }
                } else {
                    uint16_t* dst = static_cast<uint16_t*>(a.y) + (size_t)m * a.ldy + n0;
                    if (a.vec && n0 + CW <= a.N) {
#pragma unroll
                        for (int c = 0; c < CW; c += 8)
                            *reinterpret_cast<uint4*>(dst + c) =
                                make_uint4(pack_bf16x2(acc[c], acc[c + 1]), pack_bf16x2(acc[c + 2], acc[c + 3]),
                                           pack_bf16x2(acc[c + 4], acc[c + 5]), pack_bf16x2(acc[c + 6], acc[c + 7]));
                    } else {
#pragma unroll
                        for (int c = 0; c < CW; c++)
                            if (n0 + c < a.N) dst[c] = f32_to_bf16_bits(acc[c]);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(NB * BN) : "memory");
    }
    if (a.ks > 1) {
        // one tile per cluster: CTA `rank` adds columns rank, rank + ks, ...
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        float* part = reinterpret_cast<float*>(smem_raw + (smem0 - (uint32_t)__cvta_generic_to_shared(smem_raw)));
        const long long t = blockIdx.x / a.ks;
        const int m0 = (int)(t % a.mt) * kRows, n0 = (int)(t / a.mt) * BN;
        const int rows = min(kRows, a.M - m0), cols = min(BN, a.N - n0);
        const int share = (cols + a.ks - 1) / a.ks, c0 = rank * share, nc = min(share, cols - c0);
        for (int i = threadIdx.x; i < rows * nc; i += blockDim.x) {
            const int row = i / nc, c = c0 + i - row * nc;
            float v = 0.f;
            for (int q = 0; q < a.ks; q++) v += *cluster.map_shared_rank(&part[c * 129 + row], q);
            const size_t at = (size_t)(m0 + row) * a.ldy + n0 + c;
            if (a.y_f32) static_cast<float*>(a.y)[at] = v;
            else static_cast<uint16_t*>(a.y)[at] = f32_to_bf16_bits(v);
        }
        cluster.sync();  // this CTA's partial stays until its peers have read it
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)p;
    });
    return fn;
}

// Codes [rows][ld] as {128 k, box_rows} boxes; k >= K and rows past the
// matrix read as zeros.
int codes_map(const uint8_t* p, int64_t rows, int64_t K, int64_t ld, int box_rows, CUtensorMap* out) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(RENG_E_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)p, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RENG_E_CUDA, "cuTensorMapEncodeTiled (codes) failed (" + std::to_string((int)r) + ")");
    return RENG_OK;
}

constexpr size_t kSmemMax = 227 * 1024 - 1024;  // dynamic shared memory of a CTA, beside its barriers

template <int BN, int EW, int NB>
int launch_tile(const CUtensorMap& xm, const CUtensorMap& wm, Fp8Gemm& a, int grid, cudaStream_t st) {
    const size_t stage = (size_t)(a.mbox + BN) * kBK;
    a.stages = (int)std::min<size_t>(kMaxStages, (kSmemMax - 1024) / stage);
    size_t smem = a.stages * stage + 1024;
    // the last x stage is read 128 rows deep; a split leaves [BN][129] partials
    smem = std::max(smem, (size_t)1024 + (size_t)(a.stages - 1) * a.mbox * kBK + kRows * kBK);
    if (a.ks > 1) smem = std::max(smem, (size_t)1024 + (size_t)BN * 129 * 4);
    static std::once_flag once[16];
    static cudaError_t prep[16] = {};
    int dev = 0;
    RENG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16) return fail(RENG_E_UNSUPPORTED, "reng_gemm_fp8_blocks: device ordinal above 15");
    std::call_once(once[dev], [&] {
        prep[dev] = cudaFuncSetAttribute(k_gemm_fp8<BN, EW, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)kSmemMax);
    });
    RENG_CUDA_TRY(prep[dev]);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(64 + 32 * EW);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.ks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.ks > 1 ? 2 : 1;
    RENG_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_gemm_fp8<BN, EW, NB>, xm, wm, a));
    return RENG_OK;
}

}  // namespace

int gemm_fp8_blocks(const uint8_t* x, int64_t ldx, const float* sx, int64_t ldsx, int x_fmt, const uint8_t* w,
                    int64_t ldw, const float* sw, int64_t ldsw, int w_fmt, int M, int N, int K, void* y, int y_type,
                    int64_t ldy, int* err, cudaStream_t st) {
    int sms = 0;
    RENG_CUDA_TRY(current_sms(&sms));
    Fp8Gemm a{};
    a.sx = sx;
    a.sw = sw;
    a.y = y;
    a.ldsx = ldsx;
    a.ldsw = ldsw;
    a.ldy = ldy;
    a.M = M;
    a.N = N;
    a.kb = (K + kBK - 1) / kBK;
    a.mt = (M + kRows - 1) / kRows;
    a.mbox = std::min(kRows, (M + 7) / 8 * 8);
    a.y_f32 = y_type == RENG_TYPE_F32;
    a.vec = ops_aligned(y, ldy * (a.y_f32 ? 4 : 2), 16);
    a.err = err;
    // E4M3 is operand type 0, E5M2 1; f32 accumulation
    const int BN = a.mt * ((N + 255) / 256) >= sms ? 256 : (a.mt * ((N + 127) / 128) >= sms ? 128 : 64);
    a.idesc = (1u << 4) | ((uint32_t)(x_fmt == RENG_FP8_E5M2) << 7) | ((uint32_t)(w_fmt == RENG_FP8_E5M2) << 10) |
              ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
    a.nt = (N + BN - 1) / BN;
    a.ks = 1;
    const long long tiles = (long long)a.mt * a.nt;
    if (BN == 64)
        while (a.ks < kMaxSplit && tiles * a.ks * 2 <= sms && a.ks * 2 <= a.kb) a.ks *= 2;
    CUtensorMap xm, wm;
    int rc = codes_map(x, M, K, ldx, a.mbox, &xm);
    if (!rc) rc = codes_map(w, N, K, ldw, BN, &wm);
    if (rc) return rc;
    const int grid = a.ks > 1 ? (int)tiles * a.ks : (int)std::min<long long>(tiles, sms);
    if (BN == 256) return launch_tile<256, 8, 2>(xm, wm, a, grid, st);
    if (BN == 128) return launch_tile<128, 8, 4>(xm, wm, a, grid, st);
    return launch_tile<64, 4, 2>(xm, wm, a, grid, st);
}

}  // namespace reng

using namespace reng;

extern "C" int reng_gemm_fp8_blocks(const uint8_t *x, int64_t ldx, const float *x_scales, int64_t ldsx, int x_fmt,
                                    const uint8_t *w, int64_t ldw, const float *w_scales, int64_t ldsw, int w_fmt,
                                    int64_t M, int64_t N, int64_t K, void *y, int y_type, int64_t ldy, void *stream) {
    const std::string f = "reng_gemm_fp8_blocks: ";
    constexpr int64_t kMax = (int64_t)1 << 30;
    RENG_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && M <= kMax && N <= kMax && K <= kMax,
                   f + "M >= 0, N >= 1, K >= 1, each at most 2^30, not " + std::to_string(M) + " x " +
                       std::to_string(N) + " x " + std::to_string(K));
    RENG_CHECK_ARG((x_fmt == RENG_FP8_E4M3 || x_fmt == RENG_FP8_E5M2) &&
                       (w_fmt == RENG_FP8_E4M3 || w_fmt == RENG_FP8_E5M2),
                   f + "unknown format");
    RENG_CHECK_ARG(y_type == RENG_TYPE_BF16 || y_type == RENG_TYPE_F32, f + "unknown output type");
    const int64_t kb = ops_groups(K);
    RENG_CHECK_ARG(ops_pitch_ok(M, K, ldx) && ops_pitch_ok(N, K, ldw) && ops_pitch_ok(M, kb, ldsx) &&
                       ops_pitch_ok((N + 127) / 128, kb, ldsw) && ops_pitch_ok(M, N, ldy),
                   f + "a row pitch below its row, or sizes above 2^40 elements");
    if (M == 0) return RENG_OK;
    RENG_CHECK_ARG(x && x_scales && w && w_scales && y, f + "NULL buffer");
    // a single row has no pitch to keep
    if (M == 1) ldx = (ldx + 15) / 16 * 16;
    if (N == 1) ldw = (ldw + 15) / 16 * 16;
    RENG_CHECK_ARG(ops_aligned(x, ldx, 16) && ops_aligned(w, ldw, 16),
                   f + "codes must start on 16 bytes and have a row pitch that is a multiple of 16");
    RENG_CHECK_ARG(ops_aligned(x_scales, 0, 4) && ops_aligned(w_scales, 0, 4) &&
                       ops_aligned(y, 0, y_type == RENG_TYPE_F32 ? 4 : 2),
                   f + "a buffer is not aligned to its element");
    return gemm_fp8_blocks(x, ldx, x_scales, ldsx, x_fmt, w, ldw, w_scales, ldsw, w_fmt, (int)M, (int)N, (int)K, y,
                           y_type, ldy, nullptr, (cudaStream_t)stream);
}

extern "C" int reng_gemm_fp8_blocks_status(void) {
    int v = 0;
    RENG_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_fp8_gemm_err, sizeof(v)));
    if (v == 0) return RENG_OK;
    const int zero = 0;
    RENG_CUDA_TRY(cudaMemcpyToSymbol(g_fp8_gemm_err, &zero, sizeof(zero)));
    return fail(v, "reng_gemm_fp8_blocks: a product gave up on a bounded wait; its results are invalid");
}
