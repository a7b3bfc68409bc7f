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
    bool wide;                                    // rows of out (and of pre) are whole aligned vectors of a lane's outputs
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
__device__ __forceinline__ void mt_load(uint32_t from, float (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                   "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                   "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
                   "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
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
// ---- sums to outputs ----------------------------------------------------------------------------------------------------------------------
// A thread's lane of the accumulator is value p, columns are rows of out.  Eight warps read it: two have the same lanes and take 32 columns in
// turn.
__device__ __forceinline__ void mt_free(const MtPart &P, uint32_t free_, int lane) {       // this warp's columns are read: the issuer may have them back
    mt_fence_before();
    __syncwarp();
    if (lane == 0) mt_arrive(free_, P);
}

// Gradient: straight from the accumulator, while the products go on in the other one.
__device__ __forceinline__ void mt_epilogue(const MxTileArgs &A, const MtPart &P, uint32_t tmem, uint32_t done, uint32_t free_, int *dead, int warp, int lane) {
    const int quarter = warp & 3, half = (warp - kMtEpilogue) >> 2;
    int buf = 0;
    uint32_t phase = 0u;
    pdl_wait();                                                              // outputs may be what the previous kernel reads
    for (int tile = P.tile0; tile < P.tiles; tile += P.step) {
        const int n0 = tile / A.pairs_p * A.nt, cols = min(A.nt, A.rows - n0), m = 128 * (2 * (tile % A.pairs_p) + static_cast<int>(P.half)) + quarter * 32 + lane;
        const bool live = m < A.outs;
        mx_wait(done + 8 * buf, phase, dead, 24);
        mt_fence_after();
        const uint32_t from = tmem + buf * kMtRows + (static_cast<uint32_t>(quarter) << 21);
        if (32 * half >= cols) mt_free(P, free_ + 8 * buf, lane);
        for (int c = 32 * half; c < cols; c += 64) {
            float v[32];
            mt_load(from + c, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (c + 64 >= cols) mt_free(P, free_ + 8 * buf, lane);
            if (!live) continue;
            uint16_t *to = A.out + static_cast<int64_t>(n0 + c) * A.outs + m;
            if (c + 32 <= cols) {
#pragma unroll
                for (int i = 0; i < 32; i++, to += A.outs) *to = f32_to_bf16_rn(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 32; i++, to += A.outs)
                    if (c + i < cols) *to = f32_to_bf16_rn(v[i]);
            }
        }
        if (++buf == A.buffers) buf = 0, phase ^= 1u;
    }
}

// Forward, and where several pairs share the tile's c: the sums first go to shared memory as [column][lane], 128 KB for 256 rows in some 0.6 us, and the
// products go on while outputs are made of them, whole vectors a lane.  (Read straight from a lone accumulator, the next tile's products waited
// for all stores: gated 12288 x 4096, 2048 rows 310 against 257 us, with the projections kept 354 against 275.)
__device__ __forceinline__ void mt_spill(const MxTileArgs &A, uint32_t from, int cols, float *sums, int warp, int lane) {
    const int quarter = warp & 3, half = (warp - kMtEpilogue) >> 2;
    for (int c = 32 * half; c < cols; c += 64) {
        float v[32];
        mt_load(from + c + (static_cast<uint32_t>(quarter) << 21), v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32; i++) sums[(c + i) * 128 + quarter * 32 + lane] = v[i];
    }
}

__device__ __forceinline__ void mt_load_shared(const float *from, float (&v)[4]) {
    const float4 q = *reinterpret_cast<const float4 *>(from);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
}
__device__ __forceinline__ void mt_load_shared(const float *from, float (&v)[2]) {
    const float2 q = *reinterpret_cast<const float2 *>(from);
    v[0] = q.x, v[1] = q.y;
}
__device__ __forceinline__ void mt_load_cluster(uint32_t from, float (&v)[4]) {
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(from) : "memory");
}
__device__ __forceinline__ void mt_load_cluster(uint32_t from, float (&v)[2]) {
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(from) : "memory");
}

// Outputs from the sums in shared memory.  A warp takes a whole column, a lane four neighbours of it (gated: two gates, lanes 0 .. 63 of the
// accumulator, and their ups, lanes 64 .. 127).  kJoin: every pair takes each splits-th column and adds up the pairs' sums, in their order.
template <bool kGated, bool kJoin>
__device__ __forceinline__ void mt_outputs(const MxTileArgs &A, const MtPart &P, int tile, const float *sums, int warp, int lane) {
    constexpr int V = kGated ? 2 : 4, kAtOnce = 2;                           // columns that are under way together
    const int p = 2 * (tile % A.pairs_p) + static_cast<int>(P.half), n0 = tile / A.pairs_p * A.nt, cols = min(A.nt, A.rows - n0);
    const int m = (kGated ? 64 : 128) * p + V * lane, live = min(V, A.outs - m);
    float bias[V] = {}, bias_up[V] = {};
    if (A.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (i >= live) break;
            bias[i] = __uint_as_float(static_cast<uint32_t>(load_written(A.bias + m + i)) << 16);
            if (kGated) bias_up[i] = __uint_as_float(static_cast<uint32_t>(load_written(A.bias + A.outs + m + i)) << 16);
        }
    }
    const int splits = kJoin ? A.splits : 1, stride = 8 * splits;
    for (int c0 = (warp - kMtEpilogue) * splits + (kJoin ? static_cast<int>(P.pair) : 0); c0 < cols; c0 += kAtOnce * stride) {
        float v[kAtOnce][V], u[kAtOnce][V];
        const float *own = sums + V * lane;
        for (int q = 0; q < splits; q++) {
            float x[kAtOnce][V], y[kAtOnce][V];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {                              // past the last column: that one, not stored
                const int at = min(c0 + i * stride, cols - 1) * 128;
                if constexpr (kJoin) {
                    const uint32_t from = mt_peer(smem_addr(own + at), 2u * q + P.half);
                    mt_load_cluster(from, x[i]);
                    if constexpr (kGated) mt_load_cluster(from + 256, y[i]);
                } else {
                    mt_load_shared(own + at, x[i]);
                    if constexpr (kGated) mt_load_shared(own + at + 64, y[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    v[i][j] = q == 0 ? x[i][j] : v[i][j] + x[i][j];
                    if constexpr (kGated) u[i][j] = q == 0 ? y[i][j] : u[i][j] + y[i][j];
                }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const int col = c0 + i * stride;
            if (col >= cols) break;
            const int64_t row = n0 + col;
            float h[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                v[i][j] += bias[j];
                if constexpr (kGated) u[i][j] += bias_up[j];
                h[j] = kGated ? mx_act(A.activation, v[i][j]) * u[i][j] : v[i][j];
            }
            uint16_t *to = A.out + row * A.outs + m;
            float *pre = kGated && A.pre != nullptr ? A.pre + row * 2 * A.outs + m : nullptr;
            if (A.wide) {                                                    // whole vectors: all of it lives, or nothing
                if (live <= 0) continue;
                if constexpr (kGated) {
                    *reinterpret_cast<uint32_t *>(to) = pack_bf16(h[0], h[1]);
                    if (pre != nullptr) {
                        *reinterpret_cast<float2 *>(pre) = make_float2(v[i][0], v[i][1]);
                        *reinterpret_cast<float2 *>(pre + A.outs) = make_float2(u[i][0], u[i][1]);
                    }
                } else {
                    *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16(h[0], h[1]), pack_bf16(h[2], h[3]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    if (j >= live) break;
                    to[j] = f32_to_bf16_rn(h[j]);
                    if (pre != nullptr) pre[j] = v[i][j], pre[A.outs + j] = kGated ? u[i][j] : 0.f;
                }
            }
        }
    }
}

__device__ __forceinline__ void mt_epilogue_barrier() { asm volatile("bar.sync 2, 256;" ::: "memory"); }

// Every tile of the pair, whose c is its own.
template <bool kGated>
__device__ __forceinline__ void mt_epilogue_staged(const MxTileArgs &A, const MtPart &P, uint32_t tmem, uint32_t done, uint32_t free_, float *sums, int *dead, int warp, int lane) {
    int buf = 0;
    uint32_t phase = 0u;
    pdl_wait();                                                              // outputs may be what the previous kernel reads, a bias what it writes
    for (int tile = P.tile0; tile < P.tiles; tile += P.step) {
        mx_wait(done + 8 * buf, phase, dead, 24);
        mt_fence_after();
        mt_spill(A, tmem + buf * kMtTwoRows, min(A.nt, A.rows - tile / A.pairs_p * A.nt), sums, warp, lane);
        mt_free(P, free_ + 8 * buf, lane);
        mt_epilogue_barrier();
        mt_outputs<kGated, false>(A, P, tile, sums, warp, lane);
        mt_epilogue_barrier();
        if (++buf == A.buffers) buf = 0, phase ^= 1u;
    }
}

// The pairs that share a tile's c (one tile a cluster): each its sums, and after a barrier of the cluster its share of the outputs.
__device__ __forceinline__ void mt_spill_part(const MxTileArgs &A, uint32_t tmem, uint32_t done, float *sums, int *dead, int warp, int lane) {
    mx_wait(done, 0u, dead, 24);
    mt_fence_after();
    mt_spill(A, tmem, A.nt, sums, warp, lane);
}
template <bool kGated>
__device__ __forceinline__ void mt_join(const MxTileArgs &A, const MtPart &P, const float *sums, int warp, int lane) {      // every warp
    mt_cluster_sync();
    if (warp < kMtEpilogue || warp >= kMtConverter) return;
    pdl_wait();
    mt_outputs<kGated, true>(A, P, P.tile0, sums, warp, lane);
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
            cp = A.W.codes + mx_code_row(m, A.W.groups) + half * 32 + static_cast<int64_t>(group0 + g) * kMxTileCodes;
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
            q1 = __ldg(reinterpret_cast<const uint4 *>(cp + 16));
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
        float *sums = reinterpret_cast<float *>(smem + A.stages * stage_bytes);
        if (A.splits == 1) mt_epilogue_staged<kGated>(A, P, tmem, done, free_, sums, &dead, warp, lane);
        else mt_spill_part(A, tmem, done, sums, &dead, warp, lane);
    }
    if (A.splits > 1) mt_join<kGated>(A, P, reinterpret_cast<float *>(smem + A.stages * stage_bytes), warp, lane);
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
            cp = A.W.codes + at * kMxTileCodes + t * 16 + (row & 15) * kMxRowCodes;
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
        if (A.splits == 1) mt_epilogue(A, P, tmem, done, free_, &dead, warp, lane);
        else mt_spill_part(A, tmem, done, reinterpret_cast<float *>(smem), &dead, warp, lane);      // the ring's time is over
    }
    if (A.splits > 1) mt_join<false>(A, P, reinterpret_cast<float *>(smem), warp, lane);
    mt_end(tmem, &dead, warp);
}

}  // namespace bhi
