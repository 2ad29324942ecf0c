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
// Tile: 128 token rows (the MMA's M, one TMEM lane each) x bn weight rows
// (its N, a multiple of 32 up to 256 chosen per call).  A lane's scale is one
// value for all columns of a weight block, so the step out of TMEM is one FMA
// per element.  Both operands are copied by TMA as {128 k, rows} boxes with
// the 128-byte swizzle, which is the K-major operand layout; rows and columns
// past the matrix read as zeros.
// Roles (384 threads): warp 0 copies, warp 1 owns TMEM and issues the MMAs,
// warps 4-11 hold the accumulators (a warp reads the TMEM lanes of its
// quarter, warp % 4, and one half of the columns; 128 accumulators a thread,
// so the copy warps hand them their registers).  The MMAs of block b + 1 run
// into the other TMEM buffer while block b's sum is added.
//   * Many rows (PAIR): two CTAs of a cluster multiply one 256-row tile with
//     tcgen05 cta_group::2; each loads its own 128 token rows and half of the
//     weight rows, so the bytes an SM takes from L2 per block drop from 48 to
//     32 KB at bn = 256.  A block takes some 670 cycles, 512 of them the
//     MMAs', and a tile 3100 more (8192 x 28672 x 4096 1.208 M cycles, 771 a
//     block in all; 8192 x 4096 x 14336 0.548 M, 699).  The clock is the power
//     limit's: 803 us at 1.50 GHz in a first launch (2.4 PFLOP/s), 937 at 1.29
//     after a thousand, the cycles the same.
//     (The two halves of the columns as MMAs of their own read the token rows
//     twice from shared memory: 8192 x 4096 x 14336 440 us against 390.)
//   * The last round of tiles over the SMs is rarely full: it takes narrower
//     tiles than the rounds before it (1001 x 5120 x 27648: 166 us in tiles of
//     192 columns, 150 in 18 of 256 and 8 of 64; 5789 x 909 x 4011 64 and 50).
//   * Few tiles (decode): K is split over the CTAs of a cluster.  Each CTA owns
//     a share of the columns; all of them write their f32 partials of it into
//     its shared memory (stores to a peer do not wait, loads from one take a
//     microsecond), and it adds them in rank order, so the result does not
//     depend on arrival order and no workspace is needed.
// Every wait is bounded (tc.cuh); one that runs out records RENG_E_TIMEOUT in
// a device word, and the call's results are invalid.
#include <cooperative_groups.h>
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <string>

#include "fp8_encode.cuh"
#include "ops.cuh"
#include "ring.h"
#include "tc.cuh"

namespace reng {
using namespace tc;

int gemv_fp8_blocks(const uint8_t* x, int64_t ldx, const float* sx, int64_t ldsx, int x_fmt, const uint8_t* w,
                    int64_t ldw, const float* sw, int64_t ldsw, int w_fmt, int M, int N, int K, void* y, int y_type,
                    int64_t ldy, cudaStream_t st);

namespace {

// Weight elements up to which gemv_fp8.cu runs calls of at most 8, and of 9 to
// 16, token rows.  Measured on B200 (us, that kernel against this one): 8 rows
// 6144 x 4096 7.2 / 11.3, 4096 x 14336 13.5 / 17.9, 28672 x 4096 27.2 / 22.9;
// 16 rows 4096 x 4096 7.5 / 9.5, 6144 x 4096 10.7 / 11.3, 28672 x 4096 44.7 /
// 23.2 (8192 x 2048 9.2 / 7.9: the shape counts too, by less).
constexpr int64_t kGemvElems[2] = {(int64_t)1 << 26, (int64_t)1 << 25};

constexpr int kRows = 128;       // token rows of a CTA (one TMEM lane each)
constexpr int kBK = 128;         // k of a block: one swizzled row of 8-bit codes
constexpr int kMaxBn = 256;      // TMEM columns of a buffer; two buffers fill TMEM
constexpr int kMaxStages = 12;
constexpr int kMaxSplit = 4;     // K splits of a tile (CTAs of a cluster): 1, 2 or 4
constexpr int kThreads = 384;    // a warpgroup of roles, two of accumulators
constexpr int kAccWarps = 8;
// an accumulator warp's staging for its output: 32 rows of 16 columns, 17
// apart, or (PAIR) as many swizzled 32 x 32 boxes as fit 4 KB: one of f32 or
// two of bf16 (twice that costs the pipeline a stage: 400 us against 380)
constexpr int kStageOut = 32 * 17 * 4, kStageOutPair = 4096;
constexpr int kScaleSlots = 4;   // scales in flight, 4 blocks a slot:
constexpr int kScaleSlot = kRows * 16 + 64;  // [128 rows][4] of x, [3 weight blocks][4] of w
// registers per thread after the hand-over: 128 x 40 + 256 x 232 = 384 x 168,
// the registers that the block is launched with
constexpr int kRegsRole = 40, kRegsAcc = 232;

__device__ int g_fp8_gemm_err;    // set by a product whose waits ran out
__device__ int g_fp8_gemm_taken;  // the value that a status call took from it

// Read and clear in one step: a product of another stream may set the word
// meanwhile, and is told of by the next call.
__global__ void k_take_err() { g_fp8_gemm_taken = atomicExch(&g_fp8_gemm_err, 0); }

struct Fp8Gemm {
    const float *sx, *sw;
    void* y;
    int64_t ldsx, ldsw, ldy;
    int M, N, kb;      // rows, columns, 128-k blocks
    int mt, nt, bn;    // row and column tiles, their width
    int nt1, bn2;      // column tiles of that width; those behind them are bn2 wide
    int group;         // row tiles walked before the next column tile
    int ks;            // K splits (CTAs of a cluster; 1 with PAIR)
    int stages, mbox;  // pipeline stages, token rows of an x copy
    int y_f32;         // output type
    int y_vec, y_tma;  // y's rows start on 32 bytes; y is written by tensor copies (PAIR)
    int sx_vec;        // x's scales can be copied 4 at a time
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
// One MMA of 32 k: the operands' descriptors are K-major, 128-byte swizzle
// (tc.cuh, umma_desc), given by their low words (address / 16, the only part
// that changes).
constexpr uint32_t kDescLo = 1u << 16, kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;
template <bool PAIR>
__device__ __forceinline__ void umma_f8(uint32_t tmem, uint32_t alo, uint32_t blo, uint32_t idesc, bool acc) {
    if (PAIR)
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, p;\n}\n" ::"r"(tmem),
            "r"(alo), "r"(blo), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHi)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n}\n" ::"r"(tmem),
            "r"(alo), "r"(blo), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHi)
            : "memory");
}
// Arrives at `bar` (in both CTAs of a pair) when the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
    if (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        umma_commit(bar);
}
// The address of a shared-memory object of the pair's (or split's) CTA `rank`.
__device__ __forceinline__ uint32_t map_cta(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
// A tile copy whose bytes are counted at the pair leader's barrier.
__device__ __forceinline__ void pair_g2s(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tensor_s2g(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
                 "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// At most `N` of this thread's output copies still read their staging.
template <int N>
__device__ __forceinline__ void s2g_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// The role warps run their loops whole, with one elected lane issuing: their
// addresses and descriptors then live in uniform registers, where the copy
// and MMA instructions take them (run by one lane of a divergent warp, the
// four MMAs of a block took 365 cycles to issue).
__device__ __forceinline__ bool elect_lane() {
    uint32_t p;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
    return p != 0;
}
// A bounded wait: some tries without a look at the clock (a wait is taken at
// every block, and most succeed at once), then tc.cuh's.  `bad` is sticky and
// per lane: once a wait ran out a lane waits no more and runs on through its
// loop on whatever is there, in bounds and to the same end as its warp, so
// nothing diverges at the warp-wide TMEM loads.
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, bool& bad) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n .reg .u32 n;\n mov.u32 n, 0;\n"
        "TRY: mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
        " add.u32 n, n, 1;\n setp.lt.u32 p, n, 32;\n @p bra TRY;\n setp.ne.u32 p, n, n;\n"
        "DONE: selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (!ok && !bad) bad = !bar_wait(bar, parity);
}
// A product's wait for an arrival that never comes.
__global__ void k_wait_check() {
    __shared__ __align__(8) unsigned long long never;
    const uint32_t bar = (uint32_t)__cvta_generic_to_shared(&never);
    if (threadIdx.x == 0) bar_init(bar, 1);
    __syncwarp();
    bool bad = false;
    wait(bar, 0, bad);
    if (bad) atomicExch(&g_fp8_gemm_err, RENG_E_TIMEOUT);
}
// The answer to a wait takes over 100 cycles even when the phase is complete,
// so the loops ask for their next one ahead of the work between (`early`,
// which does not block) and wait only if that answer was no.
__device__ __forceinline__ uint32_t early(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok;
}
__device__ __forceinline__ void wait(uint32_t asked, uint32_t bar, uint32_t parity, bool& bad) {
    if (!asked) wait(bar, parity, bad);
}
// Lane 0's arrival, at a barrier of this CTA or (PAIR) of the pair's leader.
template <bool PAIR>
__device__ __forceinline__ void lane0_arrive(uint32_t bar, int lane) {
    if (PAIR)
        asm volatile(
            "{\n .reg .pred p;\n .reg .b32 r;\n setp.eq.s32 p, %1, 0;\n mapa.shared::cluster.u32 r, %0, 0;\n"
            " @p mbarrier.arrive.shared::cluster.b64 _, [r];\n}\n" ::"r"(bar), "r"(lane) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.eq.s32 p, %1, 0;\n @p mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(bar),
                     "r"(lane)
                     : "memory");
}
// Asynchronous copies of 16 and 4 bytes, and an arrival when this lane's are in.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float lds_f(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts_f(uint32_t addr, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// 32 bytes, a whole sector, at once.
__device__ __forceinline__ void st_global32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// The tile of index t: row tiles fastest within groups of `group`, so the
// CTAs at work together share a few row and column tiles in L2; the wide
// tiles first.
struct TileAt {
    int mi, n0, bn;
};
__device__ __forceinline__ TileAt tile_at(const Fp8Gemm& a, long long t) {
    const long long wide = (long long)a.mt * a.nt1;
    const bool second = t >= wide;
    if (second) t -= wide;
    const long long per = (long long)a.group * (second ? a.nt - a.nt1 : a.nt1);
    const int g = (int)(t / per), first = g * a.group, rows = min(a.group, a.mt - first);
    const int in = (int)(t - g * per), ni = in / rows;
    return {first + in % rows, second ? a.nt1 * a.bn + ni * a.bn2 : ni * a.bn, second ? a.bn2 : a.bn};
}

// The barriers of a CTA: operand stages, TMEM buffers and scale slots, each
// filled and free; the last MMA done.
enum : int {
    B_FULL = 0,
    B_EMPTY = B_FULL + kMaxStages,
    B_TFULL = B_EMPTY + kMaxStages,
    B_TEMPTY = B_TFULL + 2,
    B_SFULL = B_TEMPTY + 2,
    B_SEMPTY = B_SFULL + kScaleSlots,
    B_DRAIN = B_SEMPTY + kScaleSlots,
    kBars
};

// What an accumulator warp does with the blocks k0 .. k1 - 1 of a tile: NC
// chunks of 32 columns, of one weight block or (TWO) of two, the second from
// column `edge` (a multiple of 32) on.  NC 0: the warp has no outputs here and
// only keeps the barriers' count.
struct AccState {
    uint32_t tmem, bar0;     // this warp's TMEM lanes and columns; the barriers
    uint32_t sx, sw;         // scales in slot 0: this lane's row, this warp's weight block
    int lane, d, slot;       // the TMEM buffer and the scale slot of the next block
    uint32_t dph, sph;       // their phases
    bool bad;
};
template <bool PAIR, int NC, bool TWO>
__device__ __forceinline__ void add_blocks(AccState& st, int k0, int k1, int edge, f2 (&acc)[64]) {
    uint32_t td = 0, ts = 0;  // early answers for the next block's sum and the next slot of scales
    float x = 0.f, w0 = 0.f, w1 = 0.f;  // the next block's scales
    wait(st.bar0 + 8u * (B_SFULL + st.slot), st.sph, st.bad);
    if (NC > 0) {
        x = lds_f(st.sx + st.slot * kScaleSlot);
        w0 = lds_f(st.sw + st.slot * kScaleSlot);
        if (TWO) w1 = lds_f(st.sw + st.slot * kScaleSlot + 16);
    }
    for (int b = k0; b < k1; b++) {
        const float s0 = x * w0, s1 = x * w1;
        const uint32_t src = st.tmem + st.d * kMaxBn, tempty = st.bar0 + 8u * (B_TEMPTY + st.d);
        wait(td, st.bar0 + 8u * (B_TFULL + st.d), st.dph, st.bad);
        if ((st.d ^= 1) == 0) st.dph ^= 1u;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // two chunks at a time: half of the sum is read before the first
        // half is added, and the buffer is free before the second is
#pragma unroll
        for (int g = 0; g < (NC > 0 ? NC : 1); g += 2) {
            uint32_t v[2][32];
            if (NC > g) tmem_ld32(src + 32 * g, v[0]);
            if (NC > g + 1) tmem_ld32(src + 32 * g + 32, v[1]);
            if (NC > g) tmem_wait32(v[0]);
            if (NC > g + 1) tmem_wait32(v[1]);
            if (g + 2 >= NC) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                lane0_arrive<PAIR>(tempty, st.lane);
                td = early(st.bar0 + 8u * (B_TFULL + st.d), st.dph);
                const int q = (b - k0) & 3;
                if (q == 2) {
                    const int next = st.slot + 1 == kScaleSlots ? 0 : st.slot + 1;
                    ts = early(st.bar0 + 8u * (B_SFULL + next), next ? st.sph : st.sph ^ 1u);
                }
                if (q == 3 || b + 1 == k1) {
                    lane0_arrive<false>(st.bar0 + 8u * (B_SEMPTY + st.slot), st.lane);
                    if (++st.slot == kScaleSlots) st.slot = 0, st.sph ^= 1u;
                    if (b + 1 < k1) wait(ts, st.bar0 + 8u * (B_SFULL + st.slot), st.sph, st.bad);
                }
                if (NC > 0 && b + 1 < k1) {
                    const uint32_t at = st.slot * kScaleSlot + ((b + 1 - k0) & 3) * 4;
                    x = lds_f(st.sx + at);
                    w0 = lds_f(st.sw + at);
                    if (TWO) w1 = lds_f(st.sw + at + 16);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (g + h >= NC) break;
                const float s = TWO && 32 * (g + h) >= edge ? s1 : s0;
                const f2 ss = make_f2(s);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const f2 d = make_f2(__uint_as_float(v[h][2 * i]), __uint_as_float(v[h][2 * i + 1]));
                    f2& to = acc[16 * (g + h) + i];
                    to = fma_f2(d, ss, to);
                }
            }
        }
    }
}
template <bool PAIR>
__device__ __forceinline__ void add_tile(AccState& st, int nc, bool two, int k0, int k1, int edge,
                                         f2 (&acc)[64]) {
    if (nc == 0) add_blocks<PAIR, 0, false>(st, k0, k1, edge, acc);
    else if (nc == 4 && !two) add_blocks<PAIR, 4, false>(st, k0, k1, edge, acc);
    else if (nc == 4) add_blocks<PAIR, 4, true>(st, k0, k1, edge, acc);
    else if (nc == 3) add_blocks<PAIR, 3, true>(st, k0, k1, edge, acc);
    else if (nc == 2) add_blocks<PAIR, 2, true>(st, k0, k1, edge, acc);
    else add_blocks<PAIR, 1, false>(st, k0, k1, edge, acc);
}

// Every thread of the CTA (of a pair: of both) is through with TMEM.
template <bool PAIR>
__device__ __forceinline__ void cta_end() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (PAIR) cooperative_groups::this_cluster().sync();
    else __syncthreads();
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Partials of a K split: [rank of the writer][column of the owner][row].  A
// warp's 32 rows lie together, so a store to a peer is one piece of 128 bytes
// (as 32 pieces of 8 bytes a split by 4 took 9 us); a column is mbox + 1 long,
// so 32 columns of one row are read from as many banks.
//
// A thread's accumulators (row r of the tile, columns c0 .. c0 + cw - 1) into
// the shared memory of the CTAs that own the columns.
__device__ __forceinline__ void push_partials(const Fp8Gemm& a, uint32_t part, int rank, int r, int c0, int cw,
                                              const f2 (&acc)[64]) {
    const int share = a.bn / a.ks, first = c0 / share;
    const uint32_t pitch = 4u * (uint32_t)(a.mbox + 1), mine = part + (uint32_t)(rank * share) * pitch + 4u * (uint32_t)r;
    int q = first, left = share - (c0 - first * share);
    uint32_t to = (q == rank ? mine : map_cta(mine, q)) + (uint32_t)(share - left) * pitch;
#pragma unroll
    for (int i = 0; i < 64; i++) {
        if (2 * i >= cw) break;
        float lo, hi;
        split_f2(acc[i], lo, hi);
        if (q == rank) {  // its own share
            sts_f(to, lo);
            sts_f(to + pitch, hi);
        } else {
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(lo) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + pitch), "f"(hi) : "memory");
        }
        to += 2 * pitch, left -= 2;
        if (left == 0) {
            q = min(q + 1, a.ks - 1), left = share;
            to = q == rank ? mine : map_cta(mine, q);
        }
    }
}

// This CTA's share of a tile from the partials that all CTAs wrote here, in
// rank order: a warp a row, a lane a column, four rows in flight.
template <int KS>
__device__ __forceinline__ void add_partials(const Fp8Gemm& a, uint32_t part, int m0, int n0, int rank) {
    constexpr int kAcross = 4;
    const int share = a.bn / KS, rows = min(kRows, a.M - m0), cols = min(share, a.N - n0 - rank * share);
    const int warp = (int)(threadIdx.x >> 5) - (kThreads / 32 - kAccWarps);
    const uint32_t pitch = 4u * (uint32_t)(a.mbox + 1), step = (uint32_t)share * pitch;
    for (int c = threadIdx.x & 31; c < cols; c += 32) {
        const uint32_t from = part + (uint32_t)c * pitch;
        for (int r0 = warp; r0 < rows; r0 += kAcross * kAccWarps) {
            float v[kAcross][KS];
#pragma unroll
            for (int i = 0; i < kAcross; i++)
#pragma unroll
                for (int q = 0; q < KS; q++)  // past the last row: the last one's again, not written
                    v[i][q] = lds_f(from + q * step + 4u * (uint32_t)min(r0 + i * kAccWarps, rows - 1));
#pragma unroll
            for (int i = 0; i < kAcross; i++) {
                const int row = r0 + i * kAccWarps;
                if (row >= rows) break;
                float sum = v[i][0];
#pragma unroll
                for (int q = 1; q < KS; q++) sum += v[i][q];
                const size_t to = (size_t)(m0 + row) * a.ldy + n0 + rank * share + c;
                if (a.y_f32) static_cast<float*>(a.y)[to] = sum;
                else static_cast<uint16_t*>(a.y)[to] = (uint16_t)bf16x2(sum, 0.f);
            }
        }
    }
}

template <bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    k_gemm_fp8(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
               const __grid_constant__ CUtensorMap wmap2, const __grid_constant__ CUtensorMap ymap, const Fp8Gemm a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) unsigned long long bars[kBars];
    __shared__ uint32_t tmem_base_s;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t smem0 = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
    const uint32_t brows = PAIR ? (uint32_t)a.bn / 2 : (uint32_t)a.bn;
    const uint32_t abytes = (uint32_t)a.mbox * kBK, bbytes = brows * kBK;
    // x stages first: the MMA reads 128 rows from each, past a shorter box
    // into what follows, and the lanes of those rows are never used
    const uint32_t sA = smem0, sB = sA + (uint32_t)a.stages * abytes, sOut = sB + (uint32_t)a.stages * bbytes,
                   sScale = sOut + kAccWarps * (PAIR ? kStageOutPair : kStageOut),  // 16-byte aligned
                   sPart = sScale + kScaleSlots * kScaleSlot;
    const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
    auto bar = [bar0](int first, int i = 0) { return bar0 + 8u * (uint32_t)(first + i); };
    const bool clustered = PAIR || a.ks > 1;
    const int rank = clustered ? (int)cg::this_cluster().block_rank() : 0;
    int* const err = a.err ? a.err : &g_fp8_gemm_err;
    if (!PAIR && a.ks > 1) cluster_arrive();  // this CTA runs: its shared memory can be written

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; s++) {
            bar_init(bar(B_FULL, s), 1);
            bar_init(bar(B_EMPTY, s), 1);
        }
        for (int s = 0; s < 2; s++) {
            bar_init(bar(B_TFULL, s), 1);
            bar_init(bar(B_TEMPTY, s), PAIR ? 2 * kAccWarps : kAccWarps);
        }
        for (int s = 0; s < kScaleSlots; s++) {
            bar_init(bar(B_SFULL, s), 32);
            bar_init(bar(B_SEMPTY, s), kAccWarps);
        }
        bar_init(bar(B_DRAIN), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&tmem_base_s);
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (PAIR) cg::this_cluster().sync();  // the peer's barriers and TMEM are ready too
    else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base_s;
    pdl_wait();
    pdl_launch();

    const int split = PAIR ? 0 : rank, span = PAIR ? 2 : a.ks;  // CTAs per tile
    const int k0 = (int)((long long)split * a.kb / a.ks), k1 = (int)((long long)(split + 1) * a.kb / a.ks);
    const long long tiles = (long long)a.mt * a.nt, first = blockIdx.x / span, tstep = gridDim.x / span;
    constexpr int kTileRows_ = PAIR ? 2 * kRows : kRows;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRole));
        const bool leader = elect_lane();
        bool bad = false;
        if (warp == 0) {
            // ---- copies of the operands' codes ----
            Ring ring(a.stages);
            for (long long t = first; t < tiles && !bad; t += tstep) {
                const TileAt at = tile_at(a, t);
                const int m0 = at.mi * kTileRows_ + (PAIR ? rank * kRows : 0);
                const uint32_t nrows = PAIR ? (uint32_t)at.bn / 2 : (uint32_t)at.bn, bytes = abytes + nrows * kBK;
                const int n0 = at.n0 + (PAIR ? rank * (int)nrows : 0);
                const CUtensorMap* wm = at.bn == a.bn ? &wmap : &wmap2;
                for (int b = k0; b < k1; b++) {
                    const int s = ring.stage;
                    if (ring.full()) {
                        wait(bar(B_EMPTY, s), ring.phase ^ 1u, bad);
                        if (__any_sync(0xffffffffu, bad)) break;
                    }
                    const uint32_t xs = sA + (uint32_t)s * abytes, ws = sB + (uint32_t)s * bbytes;
                    if (leader) {
                        if (PAIR) {
                            // the leader CTA's barrier counts the bytes of both
                            if (rank == 0) bar_expect_tx(bar(B_FULL, s), 2 * bytes);
                            const uint32_t fb = map_cta(bar(B_FULL, s), 0);
                            pair_g2s(xs, &xmap, b * kBK, m0, fb);
                            pair_g2s(ws, wm, b * kBK, n0, fb);
                        } else {
                            bar_expect_tx(bar(B_FULL, s), bytes);
                            tensor_g2s(xs, &xmap, b * kBK, m0, bar(B_FULL, s));
                            tensor_g2s(ws, wm, b * kBK, n0, bar(B_FULL, s));
                        }
                    }
                    ring.fill();
                }
                bad = __any_sync(0xffffffffu, bad);
            }
            // The last fills' arrivals of this kind, newest first, until one gives up.
            auto landed = [&](int kind) {
                Ring last = ring;
                while (last.back())
                    if (!__all_sync(0xffffffffu, bar_wait(bar(kind, last.stage), last.phase))) return false;
                return true;
            };
            // After a wait that ran out the last copy into each stage lands
            // before the CTA may exit (a pair's follower is kept by the
            // cluster barrier at the end).
            if (bad && (!PAIR || rank == 0)) landed(B_FULL);
            // The last arrivals at EMPTY, which no refill waits for, come from
            // the tensor core on its own time (in a pair's follower, from the
            // leader's): they land before this shared memory may have another
            // owner.  Hidden behind the last block's additions (64 x 4096 x
            // 4096 10.0 us, 1001 x 5120 x 27648 148, as without it).
            bad = !landed(B_EMPTY) || bad;
            if (bad && leader) atomicExch(err, RENG_E_TIMEOUT);
        } else if (warp == 1 && (!PAIR || rank == 0)) {
            // ---- MMAs ----
            int s = 0, d = 0, used = 0;
            uint32_t ph = 0, dph = 0, af = 0, ae = 0;  // early answers: the stage, the buffer
            const uint32_t alo0 = kDescLo | sA >> 4, blo0 = kDescLo | sB >> 4;
            for (long long t = first; t < tiles; t += tstep) {
                const uint32_t idesc = a.idesc | (uint32_t)(tile_at(a, t).bn >> 3) << 17;
                for (int b = k0; b < k1; b++) {
                    const uint32_t alo = alo0 + ((uint32_t)s * abytes >> 4), blo = blo0 + ((uint32_t)s * bbytes >> 4);
                    const uint32_t dst = tmem + d * kMaxBn, done = bar(B_TFULL, d), gone = bar(B_EMPTY, s);
                    wait(af, bar(B_FULL, s), ph, bad);
                    if (used >= 2) wait(ae, bar(B_TEMPTY, d), dph ^ 1u, bad);
                    __syncwarp();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (leader && !bad) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) umma_f8<PAIR>(dst, alo + 2 * kk, blo + 2 * kk, idesc, kk != 0);
                        commit<PAIR>(done);
                        commit<PAIR>(gone);
                    }
                    if (++s == a.stages) s = 0, ph ^= 1u;
                    if ((d ^= 1) == 0) dph ^= 1u;
                    af = early(bar(B_FULL, s), ph);
                    ae = early(bar(B_TEMPTY, d), dph ^ 1u);
                    used = used < 2 ? used + 1 : used;
                }
            }
            // every MMA issued has completed before TMEM is freed
            if (leader) {
                if (PAIR)
                    asm volatile(
                        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar(B_DRAIN))
                        : "memory");
                else
                    umma_commit(bar(B_DRAIN));
            }
            bad = !bar_wait(bar(B_DRAIN), 0) || bad;
            if (bad) atomicExch(err, RENG_E_TIMEOUT);
            __syncwarp();
        } else if (warp == 2) {
            // ---- copies of the scales, 4 blocks at a time ----
            int slot = 0, used = 0;
            uint32_t ph = 0;
            const bool vec = a.sx_vec && (k0 & 3) == 0;
            for (long long t = first; t < tiles; t += tstep) {
                const TileAt at = tile_at(a, t);
                const int m0 = at.mi * kTileRows_ + (PAIR ? rank * kRows : 0);
                const int wb = min(at.n0 / kBK + (lane >> 2), (a.N - 1) / kBK);
                for (int b = k0; b < k1; b += 4) {
                    if (used >= kScaleSlots) wait(bar(B_SEMPTY, slot), ph ^ 1u, bad);
                    const uint32_t dst = sScale + slot * kScaleSlot;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = 32 * i + lane;
                        if (m0 + r >= a.M) break;
                        const float* src = a.sx + (size_t)(m0 + r) * a.ldsx + b;
                        if (vec && b + 4 <= k1) {
                            copy16(dst + 16 * r, src);
                        } else {
                            for (int j = 0; j < 4 && b + j < k1; j++) copy4(dst + 16 * r + 4 * j, src + j);
                        }
                    }
                    if (lane < 12 && b + (lane & 3) < k1)
                        copy4(dst + kRows * 16 + 4 * lane, a.sw + (size_t)wb * a.ldsw + b + (lane & 3));
                    copies_arrive(bar(B_SFULL, slot));
                    used = used < kScaleSlots ? used + 1 : used;
                    if (++slot == kScaleSlots) slot = 0, ph ^= 1u;
                }
            }
            if (bad) atomicExch(err, RENG_E_TIMEOUT);
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        // the end of the CTA, said by each side of the register hand-over for
        // itself: no code after it is shared
        if (!PAIR && a.ks > 1) cluster_wait();
        cta_end<PAIR>();
        if (warp == 1) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (PAIR)
                asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
            else
                asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        }
        if (!PAIR && a.ks > 1) {  // TMEM is already free: a CTA that waits for its peers here holds none
            cluster_arrive();
            cluster_wait();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsAcc));
        const int half = (warp - 4) >> 2;
        const int r = 32 * (warp & 3) + lane;
        const uint32_t out0 = sOut + (uint32_t)(warp - 4) * (PAIR ? kStageOutPair : kStageOut);
        uint32_t box = 0;  // staging box of the next output copy
        bool pushed = false;
        AccState st;
        st.bar0 = bar0;
        st.sx = sScale + 16 * r;
        st.lane = lane;
        st.d = st.slot = 0;
        st.dph = st.sph = 0;
        st.bad = false;
        for (long long t = first; t < tiles; t += tstep) {
            const TileAt at = tile_at(a, t);
            const int mw = at.mi * kTileRows_ + (PAIR ? rank * kRows : 0) + 32 * (warp & 3), m = mw + lane;
            // this warp's columns of the tile (multiples of 32)
            const int h0 = (at.bn / 2 + 31) / 32 * 32, c0 = half ? h0 : 0, cw = half ? at.bn - h0 : h0;
            const int n0 = at.n0 + c0;
            st.tmem = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + c0;
            const bool any = mw < a.M && n0 < a.N && cw > 0;  // the warp has outputs in this tile
            f2 acc[64];
#pragma unroll
            for (int c = 0; c < 64; c++) acc[c] = 0ull;
            // its columns touch at most two weight blocks; the second starts at column `edge`
            const int edge = (n0 / kBK + 1) * kBK - n0;
            st.sw = sScale + kRows * 16 + 16 * (n0 / kBK - at.n0 / kBK);
            add_tile<PAIR>(st, any ? cw / 32 : 0, edge < cw, k0, k1, edge, acc);
            if (!any) continue;
            if (!PAIR && a.ks > 1) {
                pushed = true;
                cluster_wait();  // all CTAs of the cluster run
                if (r < a.M - at.mi * kRows) push_partials(a, sPart, rank, r, c0, cw, acc);
            } else if (PAIR && a.y_tma) {
                // 32 rows x 32 columns at a time through this warp's staging
                // in the copy's swizzle; the copies run on behind the next tile
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    if (32 * g >= cw || n0 + 32 * g >= a.N) break;
                    const f2* q = acc + 16 * g;
                    if (a.y_f32) {  // 128-byte rows, one box
                        const uint32_t buf = out0;
                        if (lane == 0) s2g_wait_read<0>();
                        __syncwarp();
#pragma unroll
                        for (int ch = 0; ch < 8; ch++) {
                            float f0, f1, f2, f3;
                            split_f2(q[2 * ch], f0, f1);
                            split_f2(q[2 * ch + 1], f2, f3);
                            st_shared16(buf + lane * 128 + ((ch ^ (lane & 7)) << 4), __float_as_uint(f0), __float_as_uint(f1),
                                        __float_as_uint(f2), __float_as_uint(f3));
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) tensor_s2g(&ymap, n0 + 32 * g, mw, buf);
                    } else {  // 64-byte rows, two boxes
                        const uint32_t buf = out0 + box * 2048u;
                        box ^= 1;
                        if (lane == 0) s2g_wait_read<1>();
                        __syncwarp();
#pragma unroll
                        for (int ch = 0; ch < 4; ch++) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                float lo, hi;
                                split_f2(q[4 * ch + i], lo, hi);
                                w[i] = bf16x2(lo, hi);
                            }
                            st_shared16(buf + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4), w[0], w[1], w[2], w[3]);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) tensor_s2g(&ymap, n0 + 32 * g, mw, buf);
                    }
                }
            } else {
#pragma unroll
                for (int g = 0; g < 8; g++) {
                    // 16 columns: a lane's row in whole sectors, or (any
                    // pitch, and the matrix's last columns) by way of this
                    // warp's staging, consecutive lanes on consecutive columns
                    const int n = n0 + 16 * g;
                    if (16 * g >= cw || n >= a.N) break;
                    const f2* q = acc + 8 * g;
                    if (a.y_vec && n + 16 <= a.N) {
                        if (m < a.M) {
                            uint32_t w[16];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                float lo, hi;
                                split_f2(q[i], lo, hi);
                                if (a.y_f32) w[2 * i] = __float_as_uint(lo), w[2 * i + 1] = __float_as_uint(hi);
                                else w[i] = bf16x2(lo, hi);
                            }
                            char* dst = static_cast<char*>(a.y) + ((size_t)m * a.ldy + n) * (a.y_f32 ? 4 : 2);
                            st_global32(dst, *reinterpret_cast<const uint32_t(*)[8]>(w));
                            if (a.y_f32) st_global32(dst + 32, *reinterpret_cast<const uint32_t(*)[8]>(w + 8));
                        }
                    } else {
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            float lo, hi;
                            split_f2(q[i], lo, hi);
                            sts_f(out0 + 4 * (lane * 17 + 2 * i), lo);
                            sts_f(out0 + 4 * (lane * 17 + 2 * i + 1), hi);
                        }
                        __syncwarp();
                        const int c = lane & 15;
#pragma unroll 4
                        for (int i = lane >> 4; i < 32; i += 2) {
                            const float v = lds_f(out0 + 4 * (i * 17 + c));
                            if (mw + i < a.M && n + c < a.N) {
                                const size_t to = (size_t)(mw + i) * a.ldy + n + c;
                                if (a.y_f32) static_cast<float*>(a.y)[to] = v;
                                else static_cast<uint16_t*>(a.y)[to] = (uint16_t)bf16x2(v, 0.f);
                            }
                        }
                    }
                }
            }
        }
        if (st.bad) atomicExch(err, RENG_E_TIMEOUT);
        // the staging is read before the CTA's shared memory goes away
        if (PAIR && lane == 0) s2g_wait_read<0>();
        __syncwarp();
        if (!PAIR && a.ks > 1 && !pushed) cluster_wait();
        cta_end<PAIR>();
        if (!PAIR && a.ks > 1) {
            cluster_arrive();
            cluster_wait();  // all partials are here
            const TileAt at = tile_at(a, first);
            if (a.ks == 2) add_partials<2>(a, sPart, at.mi * kRows, at.n0, rank);
            else add_partials<4>(a, sPart, at.mi * kRows, at.n0, rank);
        }
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

// y [M][ldy] as {32 columns, 32 rows} boxes, swizzled as the warps stage them.
int y_map(void* y, bool f32, int64_t M, int64_t N, int64_t ldy, CUtensorMap* out) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(RENG_E_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    cuuint64_t strides[1] = {(cuuint64_t)ldy * (f32 ? 4 : 2)};
    cuuint32_t box[2] = {32, 32};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(out, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, y, dims,
                          strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RENG_E_CUDA, "cuTensorMapEncodeTiled (y) failed (" + std::to_string((int)r) + ")");
    return RENG_OK;
}

constexpr size_t kSmemMax = 227 * 1024 - 1024;  // dynamic shared memory of a CTA, beside its barriers

// Shared memory beside the pipeline's stages: the output's staging, the scales
// and (ks > 1) the partials.
size_t smem_beside(bool pair, int mbox, int bn, int ks) {
    return (size_t)kAccWarps * (pair ? kStageOutPair : kStageOut) + kScaleSlots * kScaleSlot +
           (ks > 1 ? (size_t)bn * (mbox + 1) * 4 : 0);
}

template <bool PAIR>
int launch_tiles(const CUtensorMap& xm, const CUtensorMap& wm, const CUtensorMap& wm2, const CUtensorMap& ym, Fp8Gemm& a,
                 int grid, cudaStream_t st) {
    const int brows = PAIR ? a.bn / 2 : a.bn;
    const size_t stage = (size_t)(a.mbox + brows) * kBK, out = smem_beside(PAIR, a.mbox, a.bn, a.ks);
    const int steps = (int)(((long long)a.mt * a.nt * (PAIR ? 2 : a.ks) + grid - 1) / grid) * ((a.kb + a.ks - 1) / a.ks);
    a.stages = (int)std::min<size_t>({(size_t)kMaxStages, (kSmemMax - 1024 - out) / stage, (size_t)std::max(steps, 2)});
    size_t smem = 1024 + a.stages * stage + out;
    // the last x stage is read 128 rows deep
    smem = std::max(smem, (size_t)1024 + (size_t)(a.stages - 1) * a.mbox * kBK + kRows * kBK);
    // a pair holds TMEM on two SMs while its CTAs wait for one another: it
    // takes all of their shared memory, so that no CTA of another launch that
    // does the same can sit beside one of them and wait the other way round
    if (PAIR) smem = kSmemMax;
    int dev = 0;
    RENG_CUDA_TRY(cudaGetDevice(&dev));
    static std::atomic<uint64_t> ready{0};  // devices whose limit is raised
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        RENG_CUDA_TRY(cudaFuncSetAttribute(k_gemm_fp8<PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
        if (dev < 64) ready.fetch_or((uint64_t)1 << dev);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = PAIR ? 2 : a.ks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR || a.ks > 1 ? 2 : 1;
    RENG_CUDA_TRY(cudaLaunchKernelEx(&cfg, k_gemm_fp8<PAIR>, xm, wm, wm2, ym, a));
    return RENG_OK;
}

// Cycles that a plan's busiest SM takes, from what launches of one round took
// on B200 (1024 rows x 18 bn x 4096 and 16384, at 1.9 GHz): a block costs about
// 357 + 2.1 bn cycles in one CTA and 315 + 2.13 bn in a pair, bn rounded up to
// 64 (the MMAs' own 2 bn and the issuing warp's waits, which they do not
// cover), and no less than its bytes at 64 a cycle from L2 and 23 from HBM
// when all SMs stream; a tile has a fixed cost, and a split 6000 (its barriers
// and additions, and what its clusters cost the launches around them) and a
// cycle for each 8 of the bytes that go to peers (64 rows x 4096 x 14336: 18.2
// us split by 4 against 34 whole; clusters of 3 and of 5 to 8 leave SMs of a
// GPC empty and took twice as long).
struct Plan {
    bool pair;
    int bn, ks;
    int nt1, bn2;  // bn2 > 0: nt1 column tiles of bn, the others of bn2
    double cost;
};
Plan plan(int M, int N, int kb, int sms) {
    Plan best{false, 256, 1, 0, 0, 1e300};
    const int mt1 = (M + kRows - 1) / kRows;
    for (int pair = 0; pair <= (M > kRows ? 1 : 0); pair++) {
        const int mt = pair ? (mt1 + 1) / 2 : mt1, slots = pair ? sms / 2 : sms, step = pair ? 64 : 32;
        // a block's cost in a launch of `rounds` rounds of `tiles` tiles, `blocks` blocks each
        auto block = [&](int bn, long long tiles, long long rounds, int blocks) {
            const int wide = (bn + 63) / 64 * 64;
            const double bytes = (std::min(M, kRows) + (pair ? bn / 2 : bn)) * (double)kBK;
            // all weights pass from HBM once; a round's share of it
            const double hbm = (double)N * kb * kBK / (23.0 * std::min<long long>(tiles, sms)) / ((double)rounds * blocks);
            return std::max({pair ? 315.0 + 2.13 * wide : 357.0 + 2.1 * wide, bytes / 64.0, hbm});
        };
        const double fixed = pair ? 1500.0 : 3000.0;
        for (int ks = 1; ks <= (pair ? 1 : std::min(kMaxSplit, kb)); ks *= 2) {
            if (ks > 1 && mt > slots / ks) break;
            for (int w = 1; w <= 6; w++) {
                // the narrowest tiles that fit w rounds of the SMs
                const long long fit = (long long)w * slots / ((long long)mt * ks);
                int bn = fit < 1 ? kMaxBn : (int)std::min<long long>(kMaxBn, ((N + fit - 1) / fit + step - 1) / step * step);
                const long long tiles = (long long)mt * ((N + bn - 1) / bn) * ks;
                const long long rounds = (tiles + slots - 1) / slots;
                if (ks > 1 && rounds > 1) continue;
                const int mbox = std::min(kRows, (M + 7) / 8 * 8);
                if (ks > 1 && smem_beside(false, mbox, bn, ks) + 3 * (size_t)(mbox + bn) * kBK > kSmemMax - 1024) continue;
                const int blocks = (kb + ks - 1) / ks;
                const double exchange = ks > 1 ? 6000.0 + 0.5 * std::min(M, kRows) * bn * (ks - 1) / ks : 0.0;
                const double cost = rounds * (blocks * block(bn, tiles, rounds, blocks) + fixed + exchange);
                if (cost < best.cost) best = {pair != 0, bn, ks, 0, 0, cost};
                if (bn <= 32) break;
            }
        }
        // wide tiles in all rounds but the last, which narrower ones fill
        for (int w = 2; w <= 6; w++) {
            for (int bn = kMaxBn; bn > step; bn -= step) {
                const int nt1 = (int)std::min<long long>((long long)(w - 1) * slots / mt, N / bn), left = N - nt1 * bn;
                const int fit = (int)(((long long)w * slots - (long long)mt * nt1) / mt);
                if (nt1 < 1 || fit < 1 || left < 1) continue;
                const int bn2 = ((left + fit - 1) / fit + step - 1) / step * step;
                if (bn2 >= bn) break;
                const long long tiles = (long long)mt * (nt1 + (left + bn2 - 1) / bn2);
                const double cost = kb * ((w - 1) * block(bn, tiles, w, kb) + block(bn2, tiles, w, kb)) + w * fixed;
                if (cost < best.cost) best = {pair != 0, bn, 1, nt1, bn2, cost};
            }
        }
    }
    return best;
}

}  // namespace

int gemm_fp8_blocks(const uint8_t* x, int64_t ldx, const float* sx, int64_t ldsx, int x_fmt, const uint8_t* w,
                    int64_t ldw, const float* sw, int64_t ldsw, int w_fmt, int M, int N, int K, void* y, int y_type,
                    int64_t ldy, int* err, cudaStream_t st) {
    if (M <= 16 && (int64_t)N * K <= kGemvElems[M > 8])
        return gemv_fp8_blocks(x, ldx, sx, ldsx, x_fmt, w, ldw, sw, ldsw, w_fmt, M, N, K, y, y_type, ldy, st);
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
    a.mbox = std::min(kRows, (M + 7) / 8 * 8);
    a.y_f32 = y_type == RENG_TYPE_F32;
    a.y_vec = ops_aligned(y, ldy * (a.y_f32 ? 4 : 2), 32);
    // a tensor copy's last columns are rounded up to 16 bytes, with zeros: not
    // into the columns behind y's in a larger matrix (2048 x 4094 x 4096 by
    // elements 33.9 us, 2048 x 4096 x 4096 by copies 32.6)
    a.y_tma = ops_aligned(y, ldy * (a.y_f32 ? 4 : 2), 16) && (int64_t)N * (a.y_f32 ? 4 : 2) % 16 == 0;
    a.sx_vec = ops_aligned(sx, ldsx * 4, 16);
    a.err = err;
    const Plan p = plan(M, N, a.kb, sms);
    a.bn = p.bn;
    a.ks = p.ks;
    const int rows = p.pair ? 2 * kRows : kRows;
    a.mt = (M + rows - 1) / rows;
    a.nt1 = p.bn2 ? p.nt1 : (N + a.bn - 1) / a.bn;
    a.bn2 = p.bn2;
    a.nt = a.nt1 + (p.bn2 ? (N - a.nt1 * a.bn + p.bn2 - 1) / p.bn2 : 0);
    a.group = std::min(a.mt, p.pair ? 8 : 16);
    // E4M3 is operand type 0, E5M2 1; f32 accumulation
    a.idesc = (1u << 4) | ((uint32_t)(x_fmt == RENG_FP8_E5M2) << 7) | ((uint32_t)(w_fmt == RENG_FP8_E5M2) << 10) |
              ((uint32_t)(rows >> 4) << 24);  // the kernel adds N
    CUtensorMap xm, wm, wm2, ym{};
    int rc = codes_map(x, M, K, ldx, a.mbox, &xm);
    if (!rc) rc = codes_map(w, N, K, ldw, p.pair ? a.bn / 2 : a.bn, &wm);
    wm2 = wm;
    if (!rc && p.bn2) rc = codes_map(w, N, K, ldw, p.pair ? p.bn2 / 2 : p.bn2, &wm2);
    if (!rc && p.pair && a.y_tma) rc = y_map(y, a.y_f32, M, N, ldy, &ym);
    if (rc) return rc;
    const long long tiles = (long long)a.mt * a.nt;
    if (p.pair) return launch_tiles<true>(xm, wm, wm2, ym, a, 2 * (int)std::min<long long>(tiles, sms / 2), st);
    return launch_tiles<false>(xm, wm, wm2, ym, a, a.ks > 1 ? (int)tiles * a.ks : (int)std::min<long long>(tiles, sms), st);
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
    static std::mutex mu;  // calls share g_fp8_gemm_taken
    std::lock_guard<std::mutex> lock(mu);
    RENG_CUDA_TRY(cudaDeviceSynchronize());  // non-blocking streams too
    k_take_err<<<1, 1>>>();
    RENG_CUDA_TRY(cudaGetLastError());
    int v = 0;
    RENG_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_fp8_gemm_taken, sizeof(v)));
    if (v == 0) return RENG_OK;
    return fail(v, "reng_gemm_fp8_blocks: a product gave up on a bounded wait; its results are invalid");
}

extern "C" int reng_gemm_fp8_blocks_wait_check(void *stream) {
    k_wait_check<<<1, 32, 0, (cudaStream_t)stream>>>();
    RENG_CUDA_TRY(cudaGetLastError());
    return RENG_OK;
}
