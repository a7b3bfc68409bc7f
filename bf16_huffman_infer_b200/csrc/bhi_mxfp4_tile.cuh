// Products of 4-bit microscaled weights with many rows, and the gradients of their inputs (sm_100a: tcgen05.mma, sums in tensor memory).
//
//   out[n][p] = sum over c of B[n][c] A(p, c)      forward: p a weight row m, c a column k, B = X;  gradient: p a column k, c a weight row m, B = dY
//
// Two CTAs of a cluster, on a pair of SMs, share a tile of 256 values of p (each has 128, the lanes of its accumulator) by NT rows of B (the
// accumulator's columns), of which each brings half into its shared memory: the pair's tensor cores read both halves (cta_group::2).  On
// its own an SM would write and read all of B, 96 KB of shared memory for 192 rows and 128 values of c, 750 clocks at 128 bytes a clock, where
// the products take 768: together with everything else that made 1030.
// Sixteen warps of a CTA turn codes into BF16, exactly (a code times a power of two fits), one thread requests B by TMA, one of the pair issues the
// products, eight warps read the accumulators back.  The weight is expanded once for all rows of a
// tile, so the expansion (19 instructions for eight values) stays behind the tensor cores from some 130 rows on.
#pragma once

#include <cuda.h>      // CUtensorMap and the encode entry point's types; the driver library is not linked

#include "bhi_mxfp4.cuh"

namespace bhi {

constexpr int kMtLoader = 0, kMtIssuer = 1, kMtEpilogue = 4, kMtConverter = 12;     // warps; 2 and 3 idle
constexpr int kMtPlaces = 4;                      // groups of A in tensor memory
constexpr int kMtPlaceAt = 256;                   // their first column
constexpr int kMtTeam = 8;                        // warps of a team of converters; two teams
constexpr int kMtThreads = 32 * (kMtConverter + 2 * kMtTeam);
constexpr int kMtBox = 64;                        // values of c a TMA box
constexpr uint32_t kMtABytes = 128 * kMtBox * 2;
constexpr int kMtStagesMax = 16;
constexpr uint32_t kMtSwap = 2 * 16 * 64 * 4;         // bytes through which a gated block changes lanes
constexpr int kMtRows = 256;                      // most rows of a tile
constexpr int kMtTwoRows = 128;                   // forward: most rows of a tile with two accumulators

struct MxTileArgs {
    MxWeight W;
    const uint16_t *bias;
    uint16_t *out;
    float *pre;                                   // gated, or null
    int rows, outs;                               // of out
    int activation;
    int nt, pairs_p, tiles_n, boxes_c;            // rows of a tile (a multiple of 32), pairs of tiles along p, tiles along n, boxes of 64 values of c
    int stages;                                   // of the ring
    int buffers;                                  // accumulators
    int splits, split_boxes;                      // pairs of CTAs that share a tile's c, and the boxes of each
};

// a box into this CTA's shared memory; its bytes count at the barrier of this place in the CTA that issues the products (`bar`, by mt_peer)
__device__ __forceinline__ void mt_tma_2d(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void mt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// the same with A in tensor memory: lanes are rows, a column holds two neighbours along K
__device__ __forceinline__ void mt_mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mt_store8(uint32_t to, const uint4 &a, const uint4 &b) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(to), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}
template <int N>
__device__ __forceinline__ void mt_load(uint32_t from, float (&v)[N]) {
    static_assert(N == 16, "one width");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
                   "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(from));
}
// Whether a phase is over, without waiting: asked for the next stage before this one's products are issued, so that the answer costs no time.
__device__ __forceinline__ uint32_t mt_over(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// One lane of a converged warp.  The issuing warp runs its loop as a whole and elects a lane for the products alone: operands that the
// compiler knows to be the same in all lanes stay in uniform registers.
__device__ __forceinline__ bool mt_elect() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0u;
}
__device__ __forceinline__ void mt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Which CTA this is: its half of a pair, the pair's number among those that share a tile, and the tiles and boxes that the pair walks.  By the
// block's number, which the compiler knows to be the same in all lanes.
struct MtPart {
    uint32_t half, pair;
    int tile0, step, tiles;                       // first tile, distance to the next, tiles in all
    int box0, boxes;                              // of c
    __device__ __forceinline__ explicit MtPart(const MxTileArgs &A) {
        const uint32_t size = 2u * A.splits, rank = blockIdx.x % size;
        half = rank & 1u;
        pair = rank >> 1;
        tile0 = blockIdx.x / size;
        step = gridDim.x / size;
        tiles = A.pairs_p * A.tiles_n;
        box0 = static_cast<int>(pair) * A.split_boxes;
        boxes = min(A.split_boxes, A.boxes_c - box0);
    }
    __device__ __forceinline__ uint32_t leader() const { return pair * 2u; }         // the CTA of the cluster that issues this pair's products
};
__device__ __forceinline__ uint32_t mt_peer(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// arrives at the barriers of this place in both CTAs of the pair when the products issued so far are done
__device__ __forceinline__ void mt_commit(uint32_t bar, uint32_t pair) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3u << (2u * pair))) : "memory");
}
// Arrives at the barrier of this place in the CTA that issues the products.  What is signalled lies in this CTA's own shared or tensor memory and
// has been fenced there; a release at cluster scope would wait for every copy under way (it made the gradient three times as long).
__device__ __forceinline__ void mt_arrive(uint32_t bar, const MtPart &P) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mt_peer(bar, P.leader())) : "memory");
}
__device__ __forceinline__ void mt_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 128-byte swizzle, 8-row groups (K-major) or 8-column groups (MN-major) 1024 bytes apart; lbo in 16-byte units
__device__ __forceinline__ uint64_t mt_desc(uint32_t addr, uint32_t lbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lbo) << 16) | (static_cast<uint64_t>(64u) << 32) |
           (static_cast<uint64_t>(1u) << 46) | (static_cast<uint64_t>(2u) << 61);
}
// ---- sums to outputs: a thread's lane of the accumulator is value p, columns are rows of out --------------------------------------------
// Two warps have the same lanes and take 16 columns in turn.  kGated: lanes 0 .. 63 are gates and 64 .. 127 the ups of the same outputs; of 16
// columns the first eight become the gate lanes', the others the up lanes': each hands the other half over through shared memory.
template <bool kGated>
__device__ __forceinline__ void mt_store(const MxTileArgs &A, int64_t row, int m, float v, float u) {      // bias added; u: of a gated pair
    A.out[row * A.outs + m] = f32_to_bf16_rn(kGated ? mx_act(A.activation, v) * u : v);
}
__device__ __forceinline__ float mt_bias(const MxTileArgs &A, int m, bool up, bool live) {
    if (A.bias == nullptr || !live) return 0.f;
    return __uint_as_float(static_cast<uint32_t>(load_written(A.bias + m + (up ? A.outs : 0))) << 16);
}

template <bool kGated, int kBuffer>
__device__ __forceinline__ void mt_epilogue(const MxTileArgs &A, const MtPart &P, uint32_t tmem, uint32_t done, uint32_t free_, float *swap, int *dead, int warp, int lane) {
    const int quarter = warp & 3, half = (warp - kMtEpilogue) >> 2, lane_p = quarter * 32 + lane;
    int buf = 0;
    uint32_t phase = 0u;
    swap += half * (kMtSwap / 8);
    auto read = [&]() {                                                      // this warp's columns are read: the issuer may have them back
        mt_fence_before();
        __syncwarp();
        if (lane == 0) mt_arrive(free_ + 8 * buf, P);
    };
    pdl_wait();                                                              // outputs may be what the previous kernel reads, a bias what it writes
    for (int tile = P.tile0; tile < P.tiles; tile += P.step) {
        const int p = 2 * (tile % A.pairs_p) + P.half, n0 = tile / A.pairs_p * A.nt, cols = min(A.nt, A.rows - n0);
        const int m = kGated ? 64 * p + (lane_p & 63) : 128 * p + lane_p;
        const bool up = kGated && lane_p >= 64, live = m < A.outs;
        const float bias = mt_bias(A, m, up, live);
        mx_wait(done + 8 * buf, phase, dead, 24);
        mt_fence_after();
        const uint32_t from = tmem + buf * kBuffer + (static_cast<uint32_t>(quarter) << 21);
        if (16 * half >= cols) read();
        for (int c = 16 * half; c < cols; c += 32) {
            float v[16];
            mt_load(from + c, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (c + 32 >= cols) read();
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] += bias;
            if constexpr (!kGated) {
                if (live) {
                    uint16_t *to = A.out + static_cast<int64_t>(n0 + c) * A.outs + m;
                    if (c + 16 <= cols) {
#pragma unroll
                        for (int i = 0; i < 16; i++, to += A.outs) *to = f32_to_bf16_rn(v[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++, to += A.outs)
                            if (c + i < cols) *to = f32_to_bf16_rn(v[i]);
                    }
                }
            } else {
                if (A.pre != nullptr && live) {
                    float *to = A.pre + static_cast<int64_t>(n0 + c) * 2 * A.outs + m + (up ? A.outs : 0);
#pragma unroll
                    for (int i = 0; i < 16; i++, to += 2 * static_cast<int64_t>(A.outs))
                        if (c + i < cols) *to = v[i];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) swap[((up ? 0 : 8) + i) * 64 + (lane_p & 63)] = up ? v[i] : v[8 + i];
                asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
                const int i0 = up ? 8 : 0;
                if (live) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float other = swap[(i0 + i) * 64 + (lane_p & 63)];
                        if (c + i0 + i < cols) mt_store<true>(A, n0 + c + i0 + i, m, up ? other : v[i], up ? v[8 + i] : other);
                    }
                }
                asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
            }
        }
        if (++buf == A.buffers) buf = 0, phase ^= 1u;
    }
}

// Where several pairs share the tile's c (one tile a cluster): the sums go to shared memory as [column][lane], and after a barrier of the cluster each
// pair puts every splits-th column together, in the pairs' order.
__device__ __forceinline__ void mt_spill(const MxTileArgs &A, uint32_t tmem, uint32_t done, float *sums, int *dead, int warp, int lane) {
    const int quarter = warp & 3, half = (warp - kMtEpilogue) >> 2;
    mx_wait(done, 0u, dead, 24);
    mt_fence_after();
    for (int c = 16 * half; c < A.nt; c += 32) {
        float v[16];
        mt_load(tmem + c + (static_cast<uint32_t>(quarter) << 21), v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 16; i++) sums[(c + i) * 128 + quarter * 32 + lane] = v[i];
    }
}
template <bool kGated>
__device__ __forceinline__ void mt_join(const MxTileArgs &A, const MtPart &P, const float *sums, int warp, int lane) {
    const int w = warp - kMtEpilogue, p = 2 * (P.tile0 % A.pairs_p) + P.half, n0 = P.tile0 / A.pairs_p * A.nt, cols = min(A.nt, A.rows - n0);
    constexpr int kBlocks = kGated ? 2 : 4, kAtOnce = 8;                     // blocks of 32 lanes with outputs; columns that are under way together
    const int lane_p = w % kBlocks * 32 + lane, m = (kGated ? 64 : 128) * p + lane_p;
    const bool live = m < A.outs;
    const float bias = mt_bias(A, m, false, live), bias_up = kGated ? mt_bias(A, m, true, live) : 0.f;
    const int first = (w / kBlocks) * A.splits + P.pair, stride = 8 / kBlocks * A.splits;
    for (int c0 = first; c0 < cols; c0 += kAtOnce * stride) {
        float v[kAtOnce] = {}, u[kAtOnce] = {};
        for (int q = 0; q < A.splits; q++) {
            const uint32_t from = mt_peer(smem_addr(sums) + lane_p * 4, 2u * q + P.half);
            float x[kAtOnce], y[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {                              // past the last column: some other one, not stored
                const uint32_t at = from + min(c0 + i * stride, cols - 1) * 512;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[i]) : "r"(at) : "memory");
                if constexpr (kGated) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y[i]) : "r"(at + 256) : "memory");
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                v[i] += x[i];
                if constexpr (kGated) u[i] += y[i];
            }
        }
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const int col = c0 + i * stride;
            if (col >= cols) break;
            v[i] += bias;
            u[i] += bias_up;
            if (kGated && A.pre != nullptr) {
                float *to = A.pre + static_cast<int64_t>(n0 + col) * 2 * A.outs + m;
                to[0] = v[i];
                to[A.outs] = u[i];
            }
            mt_store<kGated>(A, n0 + col, m, v[i], u[i]);
        }
    }
}

// ---- B: a stage is kBoxes times 64 values of c of this CTA's half of a tile's rows ----------------------------------------------------------
template <int kBoxes>
__device__ __forceinline__ void mt_loader(const MxTileArgs &A, const MtPart &P, const CUtensorMap *map, uint32_t base, uint32_t stage_bytes, uint32_t full, uint32_t empty,
                                          int *dead) {
    const uint32_t box = static_cast<uint32_t>(A.nt) * 64u;
    pdl_wait();
    int slot = 0;
    uint32_t phase = 1u;
    for (int tile = P.tile0; tile < P.tiles; tile += P.step) {
        const int n0 = tile / A.pairs_p * A.nt + static_cast<int>(P.half) * (A.nt / 2);
        for (int c = 0; c < P.boxes; c += kBoxes) {
            const int boxes = min(kBoxes, P.boxes - c);
            mx_wait(empty + 8 * slot, phase, dead, 20);
            if (P.half == 0) mbar_expect_tx(full + 8 * slot, 2 * boxes * box);      // both CTAs' halves
            for (int i = 0; i < boxes; i++)
                mt_tma_2d(base + slot * stage_bytes + i * box, map, (P.box0 + c + i) * kMtBox, n0, mt_peer(full + 8 * slot, P.leader()));
            if (++slot == A.stages) slot = 0, phase ^= 1u;
        }
    }
}

__device__ __forceinline__ uint32_t mt_begin(uint32_t *tmem_slot, int warp) {        // every thread; after the barriers are initialised
    if (warp == kMtIssuer) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    mt_fence_before();
    mt_cluster_sync();                                                       // the other CTA's barriers are ready too
    mt_fence_after();
    return __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
}
__device__ __forceinline__ void mt_end(uint32_t tmem, const int *dead, int warp) {
    mt_fence_before();
    mt_cluster_sync();                                                       // nobody arrives here or reads this CTA's half any more
    if (*dead)                                                               // copies and products under way land before the memory goes
        for (int i = 0; i < 10; i++) __nanosleep(100000);
    mt_cluster_sync();
    if (warp == kMtIssuer) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---- forward: A in tensor memory ------------------------------------------------------------------------------------------------------
// A thread of a team expands half a row's group (64 values) in registers while others are being multiplied, and stores it to its lane of tensor
// memory when the products that read the place are done: the weight costs shared memory nothing, which B's way in and out fills.
// Tensor memory: 256 columns of accumulators, two of up to 128 rows or one of up to 256, and four places of 64 columns, a group each, the even
// ones one team's and the odd ones the other's.  (With two places the way from one group's last product to the next in its place, some
// 1200 clocks, showed: 20.2 us for a tile of 192 rows and 4096 columns where the products take 15.)
// kGated: 64 gate rows and the 64 up rows of the same outputs make a tile.
template <bool kGated>
__global__ void __launch_bounds__(kMtThreads, 1) mx_tile_kernel(const MxTileArgs A, const __grid_constant__ CUtensorMap bmap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMtStagesMax + 4 + 2 * kMtPlaces];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t base = smem_addr(smem), box = static_cast<uint32_t>(A.nt) * 64u, stage_bytes = 2 * box;
    const uint32_t full = smem_addr(&bars[0]), empty = smem_addr(&bars[kMtStagesMax]), done = smem_addr(&bars[2 * kMtStagesMax]), free_ = done + 16,
                   a_full = done + 32, a_empty = a_full + 8 * kMtPlaces;
    const MtPart P(A);
    const int tiles = P.tiles, step = P.step, group0 = P.box0 / 2, groups = (P.boxes + 1) / 2;      // of this pair

    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < A.stages; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(done + 8 * i, 1);
            mbar_init(free_ + 8 * i, 16);
        }
        for (int i = 0; i < kMtPlaces; i++) {
            mbar_init(a_full + 8 * i, 2 * kMtTeam);
            mbar_init(a_empty + 8 * i, 1);
        }
        mbar_fence_init();
        dead = 0;
    }
    const uint32_t tmem = mt_begin(&tmem_slot, warp);

    if (warp == kMtLoader) {
        if (lane == 0) mt_loader<2>(A, P, &bmap, base, stage_bytes, full, empty, &dead);
    } else if (warp == kMtIssuer && P.half == 0) {
        // 32-bit sums, both operands BF16 and K-major
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(A.nt >> 3) << 17) | (16u << 24);
        int slot = 0, buf = 0, place = 0;
        uint32_t phase = 0u, buf_phase = 1u, a_phase = 0u;
        uint32_t b_ok = 0u, a_ok = 0u;
        for (int tile = P.tile0; tile < tiles; tile += step) {
            mx_wait(free_ + 8 * buf, buf_phase, &dead, 21);
            mt_fence_after();
            for (int g = 0; g < groups; g++) {
                if (!a_ok) mx_wait(a_full + 8 * place, a_phase, &dead, 25);
                if (!b_ok) mx_wait(full + 8 * slot, phase, &dead, 22);
                mt_fence_after();
                const uint32_t a = tmem + kMtPlaceAt + place * 64, d = tmem + buf * kMtTwoRows, used = slot, from = place;
                const uint64_t b = mt_desc(base + slot * stage_bytes, 1);
                if (++slot == A.stages) slot = 0, phase ^= 1u;
                if (++place == kMtPlaces) place = 0, a_phase ^= 1u;
                a_ok = mt_over(a_full + 8 * place, a_phase);
                b_ok = mt_over(full + 8 * slot, phase);
                if (mt_elect()) {
#pragma unroll
                    for (int k = 0; k < 4; k++) mt_mma_ta(d, a + k * 8, b + 2 * k, idesc, g > 0 || k > 0);
                    if (2 * g + 1 < P.boxes) {
#pragma unroll
                        for (int k = 0; k < 4; k++) mt_mma_ta(d, a + 32 + k * 8, b + (box >> 4) + 2 * k, idesc, 1u);
                    }
                    mt_commit(empty + 8 * used, P.pair);
                    mt_commit(a_empty + 8 * from, P.pair);
                    if (g + 1 == groups) mt_commit(done + 8 * buf, P.pair);
                }
                __syncwarp();
            }
            if (++buf == A.buffers) buf = 0, buf_phase ^= 1u;
        }
    } else if (warp >= kMtConverter) {
        const int team = (warp - kMtConverter) / kMtTeam, quarter = warp & 3, half = ((warp - kMtConverter) >> 2) & 1, row = quarter * 32 + lane;
        const uint8_t *cp = nullptr, *sp = nullptr;
        int tile = P.tile0, g = team;
        auto rows_of = [&]() {                                               // past the end: some other row, nobody reads the results
            const int p = 2 * (tile % A.pairs_p) + static_cast<int>(P.half);
            const int m = kGated ? min(64 * p + (row & 63), A.outs - 1) + (row >= 64 ? A.outs : 0) : min(128 * p + row, A.W.M - 1);
            cp = A.W.codes + mx_code_row(m, A.W.groups) + half * 2 * kMxQuarter + static_cast<int64_t>(group0 + g) * kMxTileCodes;
            sp = A.W.scales + mx_scale_row(m, A.W.groups) + static_cast<int64_t>(group0 + g) * kMxTileScales;
        };
        auto settle = [&]() {                                                // (tile, g) with g past the tile's groups: into the next tiles
            bool moved = false;
            while (g >= groups && tile < tiles) g -= groups, tile += step, moved = true;
            return moved;
        };
        uint4 q0 = make_uint4(0u, 0u, 0u, 0u), q1 = q0;
        uint32_t s = 0u;
        auto load = [&]() {
            q0 = __ldg(reinterpret_cast<const uint4 *>(cp));
            q1 = __ldg(reinterpret_cast<const uint4 *>(cp + kMxQuarter));
            s = __ldg(reinterpret_cast<const uint32_t *>(sp));
        };
        settle();
        if (tile < tiles) {
            rows_of();
            load();
        }
        const uint32_t to = tmem + kMtPlaceAt + half * 8 + (static_cast<uint32_t>(quarter) << 21);
        int place = team;
        uint32_t phase = 1u;
        while (tile < tiles) {
            uint4 h[8];
            auto expand = [&](auto large) {
                constexpr bool kLarge = decltype(large)::value;
                uint32_t f[4];
                mx_factors<kLarge>(s, f);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    h[2 * j] = mx_word_to_bf16<kLarge>(word_of(q0, j), f[j]);
                    h[2 * j + 1] = mx_word_to_bf16<kLarge>(word_of(q1, j), f[j]);
                }
            };
            if (__any_sync(0xFFFFFFFFu, (s & 0x80808080u) != 0u)) expand(std::true_type{});
            else expand(std::false_type{});
            g += 2;
            cp += 2 * kMxTileCodes;
            sp += 2 * kMxTileScales;
            if (settle() && tile < tiles) rows_of();
            if (tile < tiles) load();
            mx_wait(a_empty + 8 * place, phase, &dead, 23);
            mt_fence_after();
#pragma unroll
            for (int j = 0; j < 4; j++) mt_store8(to + place * 64 + 16 * j, h[2 * j], h[2 * j + 1]);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            mt_fence_before();
            __syncwarp();
            if (lane == 0) mt_arrive(a_full + 8 * place, P);
            if ((place += 2) >= kMtPlaces) place = team, phase ^= 1u;
        }
    } else if (warp >= kMtEpilogue) {
        if (A.splits == 1) mt_epilogue<kGated, kMtTwoRows>(A, P, tmem, done, free_, reinterpret_cast<float *>(smem + A.stages * stage_bytes), &dead, warp, lane);
        else mt_spill(A, tmem, done, reinterpret_cast<float *>(smem), &dead, warp, lane);
    }
    if (A.splits > 1) {
        mt_cluster_sync();
        if (warp >= kMtEpilogue && warp < kMtConverter) {
            pdl_wait();
            mt_join<kGated>(A, P, reinterpret_cast<float *>(smem), warp, lane);
        }
    }
    mt_end(tmem, &dead, warp);
}

// ---- gradient: A in shared memory -------------------------------------------------------------------------------------------------------
// A stage is 64 weight rows by a group of columns.  A word of eight codes is eight neighbours along p and so one 16-byte unit of the MN-major
// form of the operand: nothing is transposed.  128-byte swizzle, stores of a quarter warp on 32 different banks.  The teams take the stages of
// the ring in turn (their number is even, so that a slot is always the same team's).
__global__ void __launch_bounds__(kMtThreads, 1) mx_grad_kernel(const MxTileArgs A, const __grid_constant__ CUtensorMap bmap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMtStagesMax + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t base = smem_addr(smem), stage_bytes = kMtABytes + static_cast<uint32_t>(A.nt) * 64u;
    const uint32_t full = smem_addr(&bars[0]), empty = smem_addr(&bars[kMtStagesMax]), done = smem_addr(&bars[2 * kMtStagesMax]), free_ = done + 16;
    const MtPart P(A);
    const int tiles = P.tiles, step = P.step;

    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < A.stages; i++) {
            mbar_init(full + 8 * i, 1 + 2 * kMtTeam);                        // B, and a team of each CTA
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(done + 8 * i, 1);
            mbar_init(free_ + 8 * i, 16);
        }
        mbar_fence_init();
        dead = 0;
    }
    const uint32_t tmem = mt_begin(&tmem_slot, warp);

    if (warp == kMtLoader) {
        if (lane == 0) mt_loader<1>(A, P, &bmap, base + kMtABytes, stage_bytes, full, empty, &dead);
    } else if (warp == kMtIssuer && P.half == 0) {
        // 32-bit sums, both operands BF16, A MN-major, B K-major
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (static_cast<uint32_t>(A.nt >> 3) << 17) | (16u << 24);
        int slot = 0, buf = 0;
        uint32_t phase = 0u, buf_phase = 1u, ok = 0u;
        for (int tile = P.tile0; tile < tiles; tile += step) {
            mx_wait(free_ + 8 * buf, buf_phase, &dead, 21);
            mt_fence_after();
            for (int c = 0; c < P.boxes; c++) {
                if (!ok) mx_wait(full + 8 * slot, phase, &dead, 22);
                mt_fence_after();
                const uint32_t d = tmem + buf * kMtRows, used = slot;
                const uint64_t a = mt_desc(base + slot * stage_bytes, 512), b = mt_desc(base + slot * stage_bytes + kMtABytes, 1);
                if (++slot == A.stages) slot = 0, phase ^= 1u;
                ok = mt_over(full + 8 * slot, phase);
                if (mt_elect()) {
#pragma unroll
                    for (int k = 0; k < kMtBox / 16; k++) mt_mma(d, a + 128 * k, b + 2 * k, idesc, c > 0 || k > 0);
                    mt_commit(empty + 8 * used, P.pair);
                    if (c + 1 == P.boxes) mt_commit(done + 8 * buf, P.pair);
                }
                __syncwarp();
            }
            if (++buf == A.buffers) buf = 0, buf_phase ^= 1u;
        }
    } else if (warp >= kMtConverter) {
        const int team = (warp - kMtConverter) / kMtTeam, t = lane & 3;
        const int row = ((warp - kMtConverter) & (kMtTeam - 1)) * 8 + ((lane >> 3) | (lane & 4));      // rows 0, 4, 1, 5, 2, 6, 3, 7
        const uint32_t to = (row >> 3) * 1024 + (row & 7) * 128;
        const int storage_tiles = (A.W.M + 15) >> 4;
        int tile = P.tile0, c = team, slot = team;
        uint32_t phase = 1u;
        // units are loaded two stages of the team ahead of their use
        uint4 q, q_next;
        uint32_t s, s_next;
        int ask_tile = tile, ask_c = c;
        const uint8_t *cp = nullptr, *sp = nullptr;
        const int64_t codes_on = static_cast<int64_t>(8) * A.W.groups * kMxTileCodes, scales_on = static_cast<int64_t>(8) * A.W.groups * kMxTileScales;
        auto place = [&]() {                                                 // of stage ask_c of ask_tile; p past the end: nobody reads the results
            while (ask_c >= P.boxes && ask_tile < tiles) ask_c -= P.boxes, ask_tile += step;
            const int64_t at = static_cast<int64_t>(4 * (P.box0 + ask_c) + (row >> 4)) * A.W.groups + min(2 * (ask_tile % A.pairs_p) + static_cast<int>(P.half), A.W.groups - 1);
            cp = A.W.codes + at * kMxTileCodes + t * kMxQuarter + (row & 15) * 16;
            sp = A.W.scales + at * kMxTileScales + (row & 15) * 4;
        };
        auto load = [&](uint4 &to_q, uint32_t &to_s) {
            to_q = make_uint4(0u, 0u, 0u, 0u);
            to_s = 0u;
            if (ask_tile < tiles && 4 * (P.box0 + ask_c) + (row >> 4) < storage_tiles) {
                to_q = __ldg(reinterpret_cast<const uint4 *>(cp));
                to_s = __ldg(reinterpret_cast<const uint32_t *>(sp));
            }
            ask_c += 2;
            cp += codes_on;
            sp += scales_on;
            if (ask_c >= P.boxes) place();
        };
        auto settle = [&]() {
            while (c >= P.boxes && tile < tiles) c -= P.boxes, tile += step;
        };
        settle();
        place();
        load(q, s);
        load(q_next, s_next);
        while (tile < tiles) {
            uint4 v[4];
            auto expand = [&](auto large) {
                constexpr bool kLarge = decltype(large)::value;
                uint32_t f[4];
                mx_factors<kLarge>(s, f);
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = mx_word_to_bf16<kLarge>(word_of(q, j), f[j]);
            };
            if (__any_sync(0xFFFFFFFFu, (s & 0x80808080u) != 0u)) expand(std::true_type{});
            else expand(std::false_type{});
            q = q_next, s = s_next;
            load(q_next, s_next);
            c += 2;
            settle();
            mx_wait(empty + 8 * slot, phase, &dead, 23);
            uint8_t *dst = smem + slot * stage_bytes + to;
#pragma unroll
            for (int j = 0; j < 4; j++) *reinterpret_cast<uint4 *>(dst + (j >> 1) * 8192 + ((((j & 1) * 4 + t) ^ (row & 7)) << 4)) = v[j];
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mt_arrive(full + 8 * slot, P);
            if ((slot += 2) >= A.stages) slot = team, phase ^= 1u;
        }
    } else if (warp >= kMtEpilogue) {
        if (A.splits == 1) mt_epilogue<false, kMtRows>(A, P, tmem, done, free_, nullptr, &dead, warp, lane);
        else mt_spill(A, tmem, done, reinterpret_cast<float *>(smem), &dead, warp, lane);
    }
    if (A.splits > 1) {
        mt_cluster_sync();
        if (warp >= kMtEpilogue && warp < kMtConverter) {
            pdl_wait();
            mt_join<false>(A, P, reinterpret_cast<float *>(smem), warp, lane);
        }
    }
    mt_end(tmem, &dead, warp);
}

}  // namespace bhi
