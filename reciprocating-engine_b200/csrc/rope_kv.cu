// The step between a q/k/v product's plain output rows and attention: biases,
// the attention scale on q, RoPE, q to its buffer, k and v into the KV cache.
// The packed bf16 and FP8 projections do this in their epilogues, whose tiles
// hold a rotation's two halves; the block-scaled product (gemm_fp8.cu) writes
// rows in checkpoint order, so its model path runs this instead
// (crates/reng-synapse/src/model.rs:2962-3040).
#include "decode.cuh"

namespace reng {

// Latency-bound: 2 (q_dim + 2 kv_dim) bytes in and as many out a row, 12 KB each
// at 4096 -> 6144, against a launch of 2-3 us (the q/k/v kind, product and this,
// takes 11.3 us at one such row and 45 us at 1024).  One CTA per row; a thread takes two neighbouring dims of both halves of a
// head (or two of v), 4 bytes an access.  The rotation is
//   y[d] = x[d] cos[d] - x[d + hd/2] sin[d],  y[d + hd/2] = x[d + hd/2] cos[d + hd/2] + x[d] sin[d + hd/2].
__global__ void __launch_bounds__(256) k_rope_kv(RopeKvArgs a) {
    const int m = blockIdx.x;
    pdl_wait();
    pdl_launch();
    const int pos = __ldcg(a.row_pos + m), slot = __ldcg(a.row_slot + m);
    if (pos >= a.cap) return;
    const int half = a.hd >> 1, pairs = half >> 1, heads = a.nq + a.n_kv, kv_dim = a.n_kv * a.hd;
    const uint16_t* x = a.qkv + (size_t)m * a.ld;
    auto two = [](const uint16_t* p) { return __ldcg(reinterpret_cast<const uint32_t*>(p)); };
    auto put = [](uint16_t* p, float lo, float hi) { *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(lo, hi); };
    for (int i = threadIdx.x; i < heads * pairs; i += blockDim.x) {
        const int h = i / pairs, d = (i - h * pairs) * 2, at = h * a.hd + d;
        const bool is_q = h < a.nq;
        const float s = is_q ? a.q_scale : 1.0f;
        const uint32_t u = two(x + at), v = two(x + at + half);
        float p0 = bf16lo(u) * s, p1 = bf16hi(u) * s, q0 = bf16lo(v) * s, q1 = bf16hi(v) * s;
        if (a.bias) {  // q's part carries the scale already
            p0 += a.bias[at], p1 += a.bias[at + 1];
            q0 += a.bias[at + half], q1 += a.bias[at + half + 1];
        }
        const float* cs = a.rope_cos + (size_t)pos * a.hd + d;
        const float* sn = a.rope_sin + (size_t)pos * a.hd + d;
        uint16_t* dst = is_q ? a.q + (size_t)m * a.nq * a.hd + at
                             : a.kcache + (((size_t)slot * a.n_kv + (h - a.nq)) * a.cap + pos) * a.hd + d;
        put(dst, p0 * cs[0] - q0 * sn[0], p1 * cs[1] - q1 * sn[1]);
        put(dst + half, q0 * cs[half] + p0 * sn[half], q1 * cs[half + 1] + p1 * sn[half + 1]);
    }
    const int v0 = heads * a.hd;
    for (int i = threadIdx.x * 2; i < kv_dim; i += blockDim.x * 2) {
        const int h = i / a.hd;
        const uint32_t u = two(x + v0 + i);
        float lo = bf16lo(u), hi = bf16hi(u);
        if (a.bias) lo += a.bias[v0 + i], hi += a.bias[v0 + i + 1];
        put(a.vcache + (((size_t)slot * a.n_kv + h) * a.cap + pos) * a.hd + (i - h * a.hd), lo, hi);
    }
}

cudaError_t launch_rope_kv(const RopeKvArgs& a, int M, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(M);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_rope_kv, a);
}

}  // namespace reng
