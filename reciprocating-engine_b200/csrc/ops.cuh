// What the standalone operators share (fp8_blocks.cu, block_norm.cu,
// gemm_fp8.cu): argument rules and the launch.
#pragma once
#include "common.cuh"

namespace reng {

inline int64_t ops_groups(int64_t cols) { return (cols + 127) / 128; }

constexpr int64_t kOpsMaxCols = (int64_t)1 << 30;  // columns are counted in 32 bits

// A row pitch that holds its row, in a matrix whose extent (and that of any
// index formed from it) stays far inside 64 bits.
inline bool ops_pitch_ok(int64_t rows, int64_t cols, int64_t ld) {
    constexpr int64_t kMax = (int64_t)1 << 40;
    return rows <= kMax && cols <= kMax && ld >= cols && ld <= kMax && (rows == 0 || ld <= kMax / rows);
}

// Whether a base and a byte pitch keep every row on an n-byte boundary.
inline bool ops_aligned(const void* p, int64_t pitch_bytes, int n) {
    return (uintptr_t)p % (uintptr_t)n == 0 && pitch_bytes % n == 0;
}

// t / d for t below 2^31 by a multiplication (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994): with
// l = ceil(log2 d) and mul = floor(2^32 (2^l - d) / d) + 1, the quotient is
// (umulhi(t, mul) + t) >> l.
struct FastDiv {
    uint32_t d, mul, shift;
    explicit FastDiv(uint32_t div = 1) : d(div), shift(0) {
        while (((uint64_t)1 << shift) < d) shift++;
        mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t div(uint32_t t) const { return (__umulhi(t, mul) + t) >> shift; }
#endif
};

// SMs of the current device.
inline cudaError_t current_sms(int* sms) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    *sms = e == cudaSuccess ? num_sms(dev) : 0;
    return e;
}

// Launch with the programmatic-serialization attribute: the kernel may start
// while its predecessor drains, and waits for it (pdl_wait) before it touches
// memory.
template <typename... P, typename... A>
cudaError_t launch_ops(void (*k)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// The block-scaled product (gemm_fp8.cu) behind reng_gemm_fp8_blocks: checked
// arguments, and the device word a wait that ran out is recorded in (null: the
// entry point's own).
int gemm_fp8_blocks(const uint8_t* x, int64_t ldx, const float* sx, int64_t ldsx, int x_fmt, const uint8_t* w,
                    int64_t ldw, const float* sw, int64_t ldsw, int w_fmt, int M, int N, int K, void* y, int y_type,
                    int64_t ldy, int* err, cudaStream_t st);

}  // namespace reng
