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
#include <atomic>
#include <cmath>
#include <string>
#include <type_traits>

#include "fp8_encode.cuh"
#include "ops.cuh"
#include "row_image.h"

namespace reng {
namespace {

enum Out : int { OUT_NONE = 0, OUT_BF16, OUT_F32, OUT_E4M3, OUT_E5M2 };

struct NormArgs {
    const void *branch, *residual, *gate;
    void *y, *h;
    float* scales;
    const float *post, *pre;
    int64_t rows, ldb, ldr, ldg, ldy, ldh, lds;
    int cols;
    int tg;  // the gate's element type (RENG_TYPE_*)
    int out;
    float scale, eps, inv_n;
};

// k_block_norm's teams and their shared memory: kSlots slots a team, each one
// row's streams.  Offsets in bytes.
constexpr int kSlots = 2;
struct Plan {
    int nw, teams;             // warps of a team, teams of a CTA
    int residual, gate, slot;  // in a slot (the branch's image at 0), and its size
};

template <int TYPE>
constexpr int kBytes = TYPE == RENG_TYPE_BF16 ? 2 : 4;

template <int TYPE, typename P>
__device__ __forceinline__ P* row_at(P* base, int64_t elems) {
    return reinterpret_cast<P*>((uintptr_t)base + elems * kBytes<TYPE>);
}

constexpr int kMaxWarps = 24;  // of a CTA (named barriers: 15 teams of more than one warp)

// The warps that share a row: a CTA holds blockDim / (32 nw) such teams, each
// on a row of its own.
struct Team {
    int nw, warp, id;  // warps of a team, this warp in it, the team in its CTA
    int turn;
    __device__ __forceinline__ explicit Team(int warps) : nw(warps), turn(0) {
        const int w = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
        id = w / nw;
        warp = w - id * nw;
    }
    __device__ __forceinline__ void wait() const {
        if (nw == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(32 * nw) : "memory");
    }
    // Sum over the team, the same bits on every thread (warps added in order).
    // `red` alternates between two rows, so one barrier is enough: a row is
    // written again only after the barrier of the other's sum.
    __device__ __forceinline__ float sum(float v, float (&red)[2][kMaxWarps]) {
        v = warp_sum(v);
        if (nw == 1) return v;
        float* r = red[turn] + id * nw;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) r[warp] = v;
        wait();
        float s = 0.f;
        for (int w = 0; w < nw; w++) s += r[w];
        return s;
    }
};

// 1 / sqrt(sum / n + eps).  The hardware's root is within 2 steps, which would
// move a whole row of y over its bf16 borders; one Newton step r + r (1 - x r^2) / 2
// with the residual formed exactly leaves half a step.
__device__ __forceinline__ float inv_rms(float sum, const NormArgs& a) {
    const float x = fmaf(sum, a.inv_n, a.eps), r = rsqrtf(x), t = x * r;
    const float e = fmaf(-fmaf(x, r, -t), r, fmaf(-t, r, 1.f)), n = fmaf(0.5f * r, e, r);
    return n == n ? n : r;  // x of 0 or infinity: the limits
}

// The 4 groups of a warp tile of one row: the first column of the lane's
// values in each of its groups.
template <int G>
struct Tile {
    int c[G];
    bool live[G];
    __device__ __forceinline__ Tile(int tile, int cols) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            c[g] = (tile * kTileGroups + lane_group<G>(g)) * kFp8Group + lane_col<G>();
            live[g] = c[g] < cols;
        }
    }
};

template <bool KEEP, int TYPE, int G>
__device__ __forceinline__ void tile_load(const void* row, const Tile<G>& t, int cols, Raw16<TYPE, G>& r) {
    if constexpr (G < 4) {
        raw_zero(r);
#pragma unroll
        for (int g = 0; g < G; g++)
            if (t.live[g]) raw_load<TYPE, KEEP>(static_cast<const char*>(row) + (uint32_t)(t.c[g] * kBytes<TYPE>), g, r);
    } else if (t.c[3] + kFp8Group <= cols) {
#pragma unroll
        for (int g = 0; g < 4; g++) raw_load<TYPE, KEEP, true>(row, t.c[g], cols, g, r);
    } else {
        raw_zero(r);
#pragma unroll
        for (int g = 0; g < 4; g++)
            if (t.live[g]) raw_load<TYPE, KEEP>(row, t.c[g], cols, g, r);
    }
}

// v *= the row's elements at the tile.
template <int TYPE, int G>
__device__ __forceinline__ void tile_mul(const void* row, const Tile<G>& t, int cols, f2 (&v)[8]) {
    Raw16<TYPE, G> r;
    f2 w[8];
    tile_load<true>(row, t, cols, r);
    raw_floats(r, w);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = mul_f2(v[i], w[i]);
}
template <int G>
__device__ __forceinline__ void tile_gate(const NormArgs& a, const void* row, const Tile<G>& t, f2 (&v)[8]) {
    if (a.tg == RENG_TYPE_BF16) tile_mul<RENG_TYPE_BF16>(row, t, a.cols, v);
    else tile_mul<RENG_TYPE_F32>(row, t, a.cols, v);
}

// The vectors that every row takes, at a tile: f = post_gain * gate (where
// the gate is one row, 1 where there is neither) and pre_gain (or 1).
template <int G>
struct Vectors {
    f2 f[8], pre[8];
    __device__ __forceinline__ Vectors(const NormArgs& a, const Tile<G>& t) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = pre[i] = make_f2(1.f);
        if (a.post) tile_mul<RENG_TYPE_F32>(a.post, t, a.cols, f);
        if (a.pre) tile_mul<RENG_TYPE_F32>(a.pre, t, a.cols, pre);
        if (a.gate && !a.ldg) tile_gate(a, a.gate, t, f);
    }
};

// y's raw form from its values, rounded to TYPE.
template <int TYPE, int G>
__device__ __forceinline__ void raw_round(const f2 (&v)[8], Raw16<TYPE, G>& r) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float lo, hi;
        split_f2(v[i], lo, hi);
        if (TYPE == RENG_TYPE_F32) {
            r.w[2 * i] = __float_as_uint(lo), r.w[2 * i + 1] = __float_as_uint(hi);
        } else {
            const uint32_t p = bf16x2(lo, hi);
            if (G < 4) r.w[i] = p;
            else r.w[2 * i] = p & 0xffffu, r.w[2 * i + 1] = p >> 16;
        }
    }
}

template <int TYPE, int G>
__device__ __forceinline__ void tile_store(void* row, const Tile<G>& t, int cols, const Raw16<TYPE, G>& r) {
    if constexpr (G < 4) {
        constexpr int n = Raw16<TYPE, G>::N / (4 * G);
#pragma unroll
        for (int g = 0; g < G; g++) {
            if (!t.live[g]) continue;
            uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(row) + (uint32_t)(t.c[g] * kBytes<TYPE>));
#pragma unroll
            for (int i = 0; i < n; i++) {
                const int k = 4 * (n * g + i);
                p[i] = make_uint4(r.w[k], r.w[k + 1], r.w[k + 2], r.w[k + 3]);
            }
        }
    } else {
        using E = std::conditional_t<TYPE == RENG_TYPE_BF16, uint16_t, uint32_t>;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int c = t.c[g] + (threadIdx.x & 31);
            E* p = static_cast<E*>(row) + c;
            if (t.c[g] + kFp8Group <= cols) {
#pragma unroll
                for (int i = 0; i < 4; i++) p[32 * i] = (E)r.w[4 * g + i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (c + 32 * i < cols) p[32 * i] = (E)r.w[4 * g + i];
            }
        }
    }
}

// y of a tile, rounded, from the branch u and the residual y:
// y + (u (r(u) scale) gate) f, the gate's row of this row or null.
template <int TB, int TR, int G>
__device__ __forceinline__ void tile_residual(const NormArgs& a, const Vectors<G>& x, const void* gate,
                                              const Tile<G>& t, float inv, const Raw16<TB, G>& u, Raw16<TR, G>& y) {
    f2 v[8], w[8];
    raw_floats(u, v);
    const f2 s = make_f2(inv * a.scale);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = mul_f2(v[i], s);
    if (gate) tile_gate(a, gate, t, v);
    raw_floats(y, w);
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = fma_f2(v[i], x.f[i], w[i]);
    raw_round(w, y);
}

template <int FMT, int G>
__device__ __forceinline__ void tile_emit_fp8(const NormArgs& a, int64_t row, const Tile<G>& t, const f2 (&h)[8]) {
    float m[G], s[G], r[G];
    bool odd;
    tile_absmax(h, m, odd);
    tile_scales<FMT>(group_max(m), s, r);
    uint32_t w[4];
    tile_codes<FMT>(h, s, r, odd, w);
    uint8_t* dst = static_cast<uint8_t*>(a.h) + row * a.ldh;
    float* scales = a.scales + row * a.lds;
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (!t.live[g]) continue;
        if (lane_first<G>()) scales[t.c[g] / kFp8Group] = s[g];
        tile_store_codes<G>(dst, t.c[g], a.cols, g, w);
    }
}

// h of a tile (whole warps: the FP8 groups shuffle).
template <int TR, int G>
__device__ __forceinline__ void tile_emit(const NormArgs& a, const Vectors<G>& x, int64_t row, const Tile<G>& t,
                                          float inv, const Raw16<TR, G>& y) {
    f2 h[8];
    raw_floats(y, h);
    const f2 n = make_f2(inv);
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = mul_f2(mul_f2(h[i], n), x.pre[i]);
    if (a.out == OUT_E4M3) {
        tile_emit_fp8<RENG_FP8_E4M3, G>(a, row, t, h);
    } else if (a.out == OUT_E5M2) {
        tile_emit_fp8<RENG_FP8_E5M2, G>(a, row, t, h);
    } else if (a.out == OUT_BF16) {
        Raw16<RENG_TYPE_BF16, G> r;
        raw_round(h, r);
        tile_store(row_at<RENG_TYPE_BF16>(a.h, row * a.ldh), t, a.cols, r);
    } else {
        Raw16<RENG_TYPE_F32, G> r;
        raw_round(h, r);
        tile_store(row_at<RENG_TYPE_F32>(a.h, row * a.ldh), t, a.cols, r);
    }
}

template <int TYPE, int G>
__device__ __forceinline__ f2 square_sum(const Raw16<TYPE, G>& r, f2 s) {
    f2 v[8];
    raw_floats(r, v);
#pragma unroll
    for (int i = 0; i < 8; i++) s = fma_f2(v[i], v[i], s);
    return s;
}
__device__ __forceinline__ float f2_sum(f2 s) {
    float lo, hi;
    split_f2(s, lo, hi);
    return lo + hi;
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                 : "memory");
}
// The first `size` of N bytes; the others are zeros.
template <int N>
__device__ __forceinline__ void copy_part(void* dst, const void* src, int size) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                     "r"(size)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                     "r"(size)
                     : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A row's image (row_image.h): its whole pieces, spread over n threads, and
// (one warp) its edges, but for an odd first element.
__device__ __forceinline__ void copy_whole(uint8_t* dst, const void* row, int bytes, int thread, int n) {
    const int lead = row_lead(row);
    const char* src = static_cast<const char*>(row) - lead;
    for (int at = 16 + thread * 16; at < row_whole(lead, bytes); at += n * 16) copy16(dst + at, src + at);
}
__device__ __forceinline__ void copy_edges(uint8_t* dst, const void* row, int bytes) {
    const int lead = row_lead(row), lane = threadIdx.x & 31;
    const char* src = static_cast<const char*>(row) - lead;
    if (lane < 4) row_word(lead, bytes, lane, [&](int o, int size) { copy_part<4>(dst + o, src + o, size); });
    if (lane == 4) row_rest(lead, bytes, [&](int o, int size) { copy_part<16>(dst + o, src + o, size); });
}

// The same of an aligned row, each lane copying what it will read itself.
template <int TYPE>
__device__ __forceinline__ void copy_own(uint8_t* dst, const void* row, const Tile<2>& t) {
#pragma unroll
    for (int g = 0; g < 2; g++) {
        if (!t.live[g]) continue;
        const uint32_t at = (uint32_t)t.c[g] * kBytes<TYPE>;
        const char* src = static_cast<const char*>(row) + at;
        copy16(dst + at, src);
        if (TYPE == RENG_TYPE_F32) copy16(dst + at + 16, src + 16);
    }
}

// A team per row, a warp per tile.  The team's next row travels to shared
// memory (cp.async) while it works on one, and the vectors that every row
// takes stay in registers, so HBM is busy while teams wait for their sums.
// Held as loads in registers instead, the next row left 15 warps an SM and
// rows of any alignment spilled: 1023 x 5120, f32 branch, gate and both norms
// 22.5 us against 14.1 (4.5 TB/s); 8192 x 4096 to FP8 65 against 56 (two thirds
// of the issue slots, the codes above all, and waits on shared memory of the 24
// warps that the registers leave); 6599 x 578 to FP8 43 against 17.
// A third slot costs wide rows their second team (5120 columns: 18.3 us).
template <int TB, int TR, int G>
__global__ void __launch_bounds__(32 * kMaxWarps, 1) k_block_norm(const NormArgs a, const Plan p) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ float red[2][kMaxWarps];
    Team team(p.nw);
    const Tile<G> t(team.warp, a.cols);
    const int64_t step = (int64_t)gridDim.x * p.teams;
    int64_t row = (int64_t)team.id * gridDim.x + blockIdx.x;
    uint8_t* slots = sm + team.id * kSlots * p.slot;
    const bool gated = a.gate && a.ldg;
    auto gate_row = [&](int64_t at) -> const void* {
        return a.tg == RENG_TYPE_BF16 ? row_at<RENG_TYPE_BF16>(a.gate, at * a.ldg)
                                      : row_at<RENG_TYPE_F32>(a.gate, at * a.ldg);
    };
    // By elements, the team's last warp (the one with the fewest columns) takes
    // the edges of the rows; its lanes 0, 1 and 2 the odd first elements of the
    // residual, the branch and the gate.
    const int lane = threadIdx.x & 31;
    const bool edges = team.warp == p.nw - 1;
    auto stream = [&](int64_t at) -> const void* {
        if (lane == 0) return row_at<TR>(a.residual, at * a.ldr);
        if (lane == 1 && a.branch) return row_at<TB>(a.branch, at * a.ldb);
        return lane == 2 && gated ? gate_row(at) : nullptr;
    };
    auto copy = [&](int64_t at, uint8_t* slot) {
        if (at < a.rows) {
            const void *u = row_at<TB>(a.branch, at * a.ldb), *r = row_at<TR>(a.residual, at * a.ldr);
            if constexpr (G == 2) {
                copy_own<TR>(slot + p.residual, r, t);
                if (a.branch) copy_own<TB>(slot, u, t);
                if (gated) {
                    if (a.tg == RENG_TYPE_BF16) copy_own<RENG_TYPE_BF16>(slot + p.gate, gate_row(at), t);
                    else copy_own<RENG_TYPE_F32>(slot + p.gate, gate_row(at), t);
                }
            } else {
                const int thread = team.warp * 32 + lane, n = 32 * p.nw;
                auto image = [&](int offset, const void* from, int bytes) {
                    copy_whole(slot + offset, from, bytes, thread, n);
                    if (edges) copy_edges(slot + offset, from, bytes);
                };
                image(p.residual, r, a.cols * kBytes<TR>);
                if (a.branch) image(0, u, a.cols * kBytes<TB>);
                if (gated) image(p.gate, gate_row(at), a.cols * (a.tg == RENG_TYPE_BF16 ? 2 : 4));
            }
        }
        copy_commit();
    };
    pdl_wait();
    pdl_launch();
#pragma unroll
    for (int i = 0; i < kSlots - 1; i++) copy(row + i * step, slots + i * p.slot);
    const Vectors<G> x(a, t);
    for (int i = 0; row < a.rows; row += step, i = i + 1 == kSlots ? 0 : i + 1) {
        uint8_t *slot = slots + i * p.slot, *next = slots + (i == 0 ? kSlots - 1 : i - 1) * p.slot;
        if constexpr (G == 2) {  // the lane's own pieces: its reads of that slot are behind it
            copy(row + (kSlots - 1) * step, next);
            copy_wait<kSlots - 1>();
        } else {  // pieces of other lanes: all of this row there, all reads of the last one done
            copy_wait<kSlots - 2>();
            // an odd first element, whose sector is in L2 with the copies
            // (carried in a register from the copies on it spilled)
            if (edges) {
                const void* from = stream(row);
                const int lead = row_lead(from);
                if (row_odd(lead))
                    *reinterpret_cast<unsigned short*>(slot + (lane == 0 ? p.residual : lane == 1 ? 0 : p.gate) + lead) =
                        *static_cast<const unsigned short*>(from);
            }
            team.wait();
            copy(row + (kSlots - 1) * step, next);
        }
        Raw16<TB, G> u;
        Raw16<TR, G> y;
        tile_load<true>(slot + p.residual + (G == 2 ? 0 : row_lead(row_at<TR>(a.residual, row * a.ldr))), t, a.cols, y);
        if (a.branch) {
            tile_load<true>(slot + (G == 2 ? 0 : row_lead(row_at<TB>(a.branch, row * a.ldb))), t, a.cols, u);
            float inv = 1.f;
            if (a.post) inv = inv_rms(team.sum(f2_sum(square_sum(u, 0ull)), red), a);
            const void* gate = gated ? slot + p.gate + (G == 2 ? 0 : row_lead(gate_row(row))) : nullptr;
            tile_residual(a, x, gate, t, inv, u, y);
            tile_store(row_at<TR>(a.y, row * a.ldy), t, a.cols, y);
        }
        if (a.out == OUT_NONE) continue;
        const float inv = inv_rms(team.sum(f2_sum(square_sum(y, 0ull)), red), a);
        tile_emit(a, x, row, t, inv, y);
    }
}

// Rows too long for shared memory: three passes over the columns, each warp
// reading back only what it wrote itself.  A thread's sum over its tiles is in
// 64 bits (one addition a tile): in f32 the mean square of 2^24 equal values
// was 920 half-steps off.
template <int TB, int TR, int G>
__global__ void __launch_bounds__(512) k_block_norm_long(const NormArgs a) {
    __shared__ float red[2][kMaxWarps];
    Team team(16);
    const int tiles = (a.cols + kTileGroups * kFp8Group - 1) / (kTileGroups * kFp8Group);
    pdl_wait();
    pdl_launch();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const void *branch = row_at<TB>(a.branch, row * a.ldb), *residual = row_at<TR>(a.residual, row * a.ldr);
        void* out = row_at<TR>(a.y, row * a.ldy);
        const void* gate = !a.gate || !a.ldg ? nullptr
                           : a.tg == RENG_TYPE_BF16 ? row_at<RENG_TYPE_BF16>(a.gate, row * a.ldg)
                                                    : row_at<RENG_TYPE_F32>(a.gate, row * a.ldg);
        float inv = 1.f;
        if (a.branch && a.post) {
            double s = 0.;
            for (int i = team.warp; i < tiles; i += team.nw) {
                Raw16<TB, G> u;
                tile_load<false>(branch, Tile<G>(i, a.cols), a.cols, u);
                s += f2_sum(square_sum(u, 0ull));
            }
            inv = inv_rms(team.sum((float)s, red), a);
        }
        double s = 0.;
        for (int i = team.warp; i < tiles; i += team.nw) {
            const Tile<G> t(i, a.cols);
            Raw16<TR, G> y;
            tile_load<false>(residual, t, a.cols, y);
            if (a.branch) {
                Raw16<TB, G> u;
                tile_load<false>(branch, t, a.cols, u);
                tile_residual(a, Vectors<G>(a, t), gate, t, inv, u, y);
                tile_store(out, t, a.cols, y);
            }
            s += f2_sum(square_sum(y, 0ull));
        }
        if (a.out == OUT_NONE) continue;
        inv = inv_rms(team.sum((float)s, red), a);
        for (int i = team.warp; i < tiles; i += team.nw) {
            const Tile<G> t(i, a.cols);
            Raw16<TR, G> y;
            tile_load<false>(a.branch ? out : residual, t, a.cols, y);
            tile_emit(a, Vectors<G>(a, t), row, t, inv, y);
        }
    }
}

// The image of a row of `cols` elements, with room for its lead.
int64_t image(int64_t cols, int esize) { return (cols * esize + 15) / 16 * 16 + 16; }

constexpr int kSmemMax = 226 * 1024;

template <int TB, int TR, int G>
cudaError_t launch_row(const NormArgs& a, int sms, cudaStream_t st) {
    constexpr int kTile = kTileGroups * kFp8Group;
    const int tiles = (int)(((int64_t)a.cols + kTile - 1) / kTile), eg = a.tg == RENG_TYPE_BF16 ? 2 : 4;
    const int64_t residual = a.branch ? image(a.cols, kBytes<TB>) : 0, gate = residual + image(a.cols, kBytes<TR>),
                  slot = gate + (a.gate && a.ldg ? image(a.cols, eg) : 0);
    if (tiles > kMaxWarps || kSlots * slot > kSmemMax)
        return launch_ops(k_block_norm_long<TB, TR, G>, dim3((unsigned)std::min<int64_t>(a.rows, (int64_t)sms * 4)),
                          dim3(512), 0, st, a);
    Plan p;
    p.nw = tiles;
    // rows go to as many SMs as there are, then to teams of one CTA
    p.teams = (int)std::min<int64_t>({p.nw == 1 ? kMaxWarps : 15, kMaxWarps / p.nw, kSmemMax / (kSlots * slot), (a.rows + sms - 1) / sms});
    p.residual = (int)residual, p.gate = (int)gate, p.slot = (int)slot;
    const size_t smem = (size_t)(p.teams * kSlots * slot);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<uint64_t> ready{0};  // devices whose limit is raised
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        e = cudaFuncSetAttribute(k_block_norm<TB, TR, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or((uint64_t)1 << dev);
    }
    const dim3 grid((unsigned)std::min<int64_t>((a.rows + p.teams - 1) / p.teams, sms));
    return launch_ops(k_block_norm<TB, TR, G>, grid, dim3((unsigned)(32 * p.teams * p.nw)), smem, st, a, p);
}

int launch(const NormArgs& a, int tb, int tr, bool vec, cudaStream_t st) {
    int sms = 0;
    RENG_CUDA_TRY(current_sms(&sms));
    constexpr int B = RENG_TYPE_BF16, F = RENG_TYPE_F32;
    auto pick = [&](auto v) {
        constexpr int V = decltype(v)::value;
        if (tr == B) return tb == B ? launch_row<B, B, V>(a, sms, st) : launch_row<F, B, V>(a, sms, st);
        return tb == B ? launch_row<B, F, V>(a, sms, st) : launch_row<F, F, V>(a, sms, st);
    };
    const cudaError_t e = vec ? pick(std::integral_constant<int, 2>()) : pick(std::integral_constant<int, 4>());
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
    RENG_CHECK_ARG(d->rows >= 0 && d->cols >= 1 && d->cols <= kOpsMaxCols, f + "rows >= 0 and cols in [1, 2^30], not " + std::to_string(d->rows) +
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
    // in place a row is written where it was read; at another pitch, where another row is still to be read
    RENG_CHECK_ARG(!d->branch || d->y != d->residual || d->rows == 1 || d->ld_y == d->ld_residual,
                   f + "y in place of residual at another row pitch");
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
    a.cols = (int)d->cols;
    a.inv_n = 1.0f / (float)d->cols;
    a.ldb = d->ld_branch;
    a.ldr = d->ld_residual;
    a.ldg = d->ld_gate;
    a.ldy = d->ld_y;
    a.ldh = d->ld_h;
    a.lds = d->ld_scales;
    const int tb = d->branch ? d->branch_type : d->residual_type, tr = d->residual_type;
    a.tg = d->gate_type;
    a.out = d->out;
    a.scale = d->scale;
    a.eps = d->eps;
    auto aligned = [](const void* p, int64_t ld, int esz, int n) { return !p || ops_aligned(p, ld * esz, n); };
    const int eb = host_esize(tb), er = host_esize(tr), eg = host_esize(a.tg);
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
    return launch(a, tb, tr, vec, (cudaStream_t)stream);
}
