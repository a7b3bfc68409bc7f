// Products of 4-bit microscaled weights with many rows, and the gradients of their inputs (sm_100a: tcgen05.mma, sums in tensor memory).
//
//   out[n][p] = sum over c of B[n][c] A(p, c)      forward: p a weight row m, c a column k, B = X;  gradient: p a column k, c a weight row m, B = dY
//
// A tile is 128 values of p (the lanes of an accumulator) by NT rows of B (its columns), walked in stages of 64 values of c.  Eight warps turn
// codes into BF16 in shared memory, exactly (a code times a power of two fits), one thread requests B by TMA, one issues the products, four warps
// read the accumulators back, two of which alternate between tiles.  The weight is expanded once for up to 256 rows, so the expansion
// (19 instructions for eight values) stays behind the tensor cores:
//   * forward, a stage is [128 rows][64 columns], K-major;  gradient, [64 rows][128 columns], which is the MN-major form of the same operand:
//     a word of eight codes is eight neighbours along k and so one 16-byte unit of either, and nothing is transposed;
//   * both with the 128-byte swizzle, stores of a quarter warp on 32 different banks.
// A code's bits s eem are moved to a BF16's sign, lowest exponent and highest mantissa bits: that is its value times 2^-126, the
// subnormal code 0.5 included, and one product by 2^(126 + s - 127) makes both the value and its scale.  Scales above 2 (2^(126 + s - 127) would
// overflow) take two products.
// kGated: 64 gate rows and 64 up rows of the same outputs make a tile; half of each accumulator block changes lanes through shared memory.
#pragma once

#include <cuda.h>      // CUtensorMap and the encode entry point's types; the driver library is not linked

#include "bhi_mxfp4.cuh"

namespace bhi {

enum MxTileKind { kMxPlain = 0, kMxGatedPair = 1, kMxGradient = 2 };

constexpr int kMtLoader = 0, kMtIssuer = 1, kMtEpilogue = 4, kMtConverter = 8;      // warps; 2 and 3 idle
constexpr int kMtConverters = 8;
constexpr int kMtThreads = 32 * (kMtConverter + kMtConverters);
constexpr int kMtStage = 64;                      // values of c
constexpr uint32_t kMtABytes = 128 * kMtStage * 2;
constexpr int kMtStagesMax = 10;
constexpr uint32_t kMtSwap = 32 * 64 * 4;         // bytes through which a gated block changes lanes

struct MxTileArgs {
    MxWeight W;
    const uint16_t *bias;
    uint16_t *out;
    float *pre;                                   // gated, or null
    int rows, outs;                               // of out
    int activation;
    int nt, tiles_p, tiles_n, stages_c;           // rows of a tile, tiles, stages of a tile
    int stages;                                   // of the ring
};

__device__ __forceinline__ void mt_tma_2d(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void mt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mt_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 128-byte swizzle, 8-row groups (K-major) or 8-column groups (MN-major) 1024 bytes apart; lbo in 16-byte units
__device__ __forceinline__ uint64_t mt_desc(uint32_t addr, uint32_t lbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lbo) << 16) | (static_cast<uint64_t>(64u) << 32) |
           (static_cast<uint64_t>(1u) << 46) | (static_cast<uint64_t>(2u) << 61);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Eight codes and their scale byte as eight BF16 values in element order.
__device__ __forceinline__ uint4 mx_word_to_bf16(uint32_t w, uint32_t s, bool large) {
    constexpr uint32_t kMag = 0x01C001C0u, kSign = 0x80008000u;
    uint32_t h[4];
    h[0] = ((w << 6) & kMag) | ((w << 12) & kSign);
    h[1] = ((w << 2) & kMag) | ((w << 8) & kSign);
    h[2] = ((w >> 2) & kMag) | ((w << 4) & kSign);
    h[3] = ((w >> 6) & kMag) | (w & kSign);
    if (!large) {
        const uint32_t f = s * 0x00800080u + 0x3F003F00u;                    // 2^(s - 1)
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = mul_bf16x2(h[i], f);
    } else {
        const uint32_t f = s == 0u ? 0x00400040u : s * 0x00800080u;          // 2^(s - 127); 255: infinity, and its codes are zero
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = mul_bf16x2(mul_bf16x2(h[i], 0x7E807E80u), f);
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
}

// A wait of at most about a second; when one runs out, the kernel's status word is set and no other wait of the CTA goes on.
__device__ __forceinline__ void mt_wait(uint32_t bar, uint32_t parity, int *dead, int status) {
    if (mbar_try_wait(bar, parity)) return;
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*static_cast<volatile int *>(dead)) return;
        if (global_ns() - t0 > 1000000000ull) {
            atomicExch(dead, 1);
            atomicExch(&g_staged_status, status);
            return;
        }
    }
}

template <int kKind>
__global__ void __launch_bounds__(kMtThreads, 1) mx_tile_kernel(const MxTileArgs A, const __grid_constant__ CUtensorMap bmap) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMtStagesMax + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = smem_addr(smem);
    const uint32_t full = smem_addr(&bars[0]), empty = smem_addr(&bars[kMtStagesMax]), done = smem_addr(&bars[2 * kMtStagesMax]), free_ = done + 16;
    const uint32_t b_bytes = static_cast<uint32_t>(A.nt) * 128u, stage_bytes = kMtABytes + b_bytes;
    const int tiles = A.tiles_p * A.tiles_n;

    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < A.stages; i++) {
            mbar_init(full + 8 * i, kMtConverters + 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(done + 8 * i, 1);
            mbar_init(free_ + 8 * i, 4);
        }
        mbar_fence_init();
        dead = 0;
    }
    if (warp == kMtIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;

    if (warp == kMtLoader) {
        if (lane == 0) {
            pdl_wait();
            int slot = 0;
            uint32_t phase = 1u;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                const int n0 = tile / A.tiles_p * A.nt;
                for (int c = 0; c < A.stages_c; c++) {
                    mt_wait(empty + 8 * slot, phase, &dead, 20);
                    mbar_expect_tx(full + 8 * slot, b_bytes);
                    mt_tma_2d(base + slot * stage_bytes + kMtABytes, &bmap, c * kMtStage, n0, full + 8 * slot);
                    if (++slot == A.stages) slot = 0, phase ^= 1u;
                }
            }
        }
    } else if (warp == kMtIssuer) {
        if (lane == 0) {
            // 32-bit sums, both operands BF16, B K-major, A K-major or (gradient) MN-major
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (kKind == kMxGradient ? 1u << 15 : 0u) | (static_cast<uint32_t>(A.nt >> 3) << 17) | (8u << 24);
            int slot = 0, buf = 0;
            uint32_t phase = 0u, buf_phase = 1u;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                mt_wait(free_ + 8 * buf, buf_phase, &dead, 21);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int c = 0; c < A.stages_c; c++) {
                    mt_wait(full + 8 * slot, phase, &dead, 22);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t a = base + slot * stage_bytes, b = a + kMtABytes;
#pragma unroll
                    for (int k = 0; k < kMtStage / 16; k++)
                        mt_mma(tmem + buf * 256, kKind == kMxGradient ? mt_desc(a + k * 2048, 512) : mt_desc(a + k * 32, 1), mt_desc(b + k * 32, 1), idesc, c > 0 || k > 0);
                    mt_commit(empty + 8 * slot);
                    if (++slot == A.stages) slot = 0, phase ^= 1u;
                }
                mt_commit(done + 8 * buf);
                if ((buf ^= 1) == 0) buf_phase ^= 1u;
            }
        }
    } else if (warp >= kMtConverter) {
        // ---- codes to BF16 ---------------------------------------------------------------------------------------------------
        const int w = warp - kMtConverter, t = lane & 3;
        const int r8 = (lane >> 3) | (lane & 4);                     // rows 0, 4, 1, 5, 2, 6, 3, 7: a quarter warp's units lie on 32 banks
        int slot = 0;
        uint32_t phase = 1u;
        auto begin = [&]() { mt_wait(empty + 8 * slot, phase, &dead, 23); };
        auto end = [&]() {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * slot);
            if (++slot == A.stages) slot = 0, phase ^= 1u;
        };
        if constexpr (kKind == kMxGradient) {
            // stage c: rows 64 c .. of the weight, group p of columns; this thread's row and quarter
            const int row = w * 8 + r8, storage_tiles = (A.W.M + 15) >> 4;
            const uint32_t to = (row >> 3) * 1024 + (row & 7) * 128;
            auto load = [&](int p, int c, uint4 &q, uint32_t &s) {
                const int tile = 4 * c + (row >> 4);
                q = make_uint4(0u, 0u, 0u, 0u);
                s = 0u;
                if (tile < storage_tiles) {
                    const int64_t at = static_cast<int64_t>(tile) * A.W.groups + p;
                    q = __ldg(reinterpret_cast<const uint4 *>(A.W.codes + at * kMxTileCodes + (row & 15) * 64 + t * 16));
                    s = __ldg(reinterpret_cast<const uint32_t *>(A.W.scales + at * kMxTileScales + (row & 15) * 4));
                }
            };
            uint4 q;
            uint32_t s;
            if (static_cast<int>(blockIdx.x) < tiles) load(blockIdx.x % A.tiles_p, 0, q, s);
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                const int p = tile % A.tiles_p;
                for (int c = 0; c < A.stages_c; c++) {
                    const uint4 now = q;
                    const uint32_t sc = s;
                    if (c + 1 < A.stages_c) load(p, c + 1, q, s);
                    else if (tile + static_cast<int>(gridDim.x) < tiles) load((tile + gridDim.x) % A.tiles_p, 0, q, s);
                    const bool large = (sc & 0x80808080u) != 0u;
                    begin();
                    uint8_t *dst = smem + slot * stage_bytes + to;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint4 v = mx_word_to_bf16(j == 0 ? now.x : j == 1 ? now.y : j == 2 ? now.z : now.w, (sc >> (8 * j)) & 255u, large);
                        *reinterpret_cast<uint4 *>(dst + (j >> 1) * 8192 + ((((j & 1) * 4 + t) ^ (row & 7)) << 4)) = v;
                    }
                    end();
                }
            }
        } else {
            // stage c: columns 64 c .. of 128 weight rows; this thread's two rows and quarter, a group (two stages) loaded at a time
            int row[2];
            row[0] = w * 8 + r8;
            row[1] = row[0] + 64;
            const uint8_t *cp[2], *sp[2];
            auto rows_of = [&](int p) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    int m;
                    if constexpr (kKind == kMxGatedPair) m = i == 0 ? min(64 * p + row[0], A.outs - 1) : A.outs + min(64 * p + row[0], A.outs - 1);
                    else m = min(128 * p + row[i], A.W.M - 1);               // past the end: nobody reads the results
                    cp[i] = A.W.codes + mx_code_row(m, A.W.groups) + t * 16;
                    sp[i] = A.W.scales + mx_scale_row(m, A.W.groups);
                }
            };
            uint4 q[2];
            uint32_t s[2];
            auto load = [&](int g) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    q[i] = __ldg(reinterpret_cast<const uint4 *>(cp[i] + static_cast<int64_t>(g) * kMxTileCodes));
                    s[i] = __ldg(reinterpret_cast<const uint32_t *>(sp[i] + static_cast<int64_t>(g) * kMxTileScales));
                }
            };
            if (static_cast<int>(blockIdx.x) < tiles) {
                rows_of(blockIdx.x % A.tiles_p);
                load(0);
            }
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                for (int c = 0; c < A.stages_c; c += 2) {
                    const uint4 now[2] = {q[0], q[1]};
                    const uint32_t sc[2] = {s[0], s[1]};
                    if (c + 2 < A.stages_c) {
                        load((c + 2) >> 1);
                    } else if (tile + static_cast<int>(gridDim.x) < tiles) {
                        rows_of((tile + gridDim.x) % A.tiles_p);
                        load(0);
                    }
                    const bool large = ((sc[0] | sc[1]) & 0x80808080u) != 0u;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (c + h >= A.stages_c) break;
                        begin();
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            uint8_t *dst = smem + slot * stage_bytes + row[i] * 128;
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const uint32_t word = h == 0 ? (j == 0 ? now[i].x : now[i].y) : (j == 0 ? now[i].z : now[i].w);
                                *reinterpret_cast<uint4 *>(dst + (((j * 4 + t) ^ (row[i] & 7)) << 4)) = mx_word_to_bf16(word, (sc[i] >> (8 * (2 * h + j))) & 255u, large);
                            }
                        }
                        end();
                    }
                }
            }
        }
    } else if (warp >= kMtEpilogue) {
        // ---- sums to outputs: this thread's lane of the accumulator is value p, columns are rows of out ---------------------------------
        const int quarter = warp & 3, lane_p = quarter * 32 + lane;
        float *swap = reinterpret_cast<float *>(smem + A.stages * stage_bytes);
        int buf = 0;
        uint32_t buf_phase = 0u;
        pdl_wait();                                                          // outputs may be what the previous kernel reads, a bias what it writes
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const int p = tile % A.tiles_p, n0 = tile / A.tiles_p * A.nt, cols = min(A.nt, A.rows - n0);
            constexpr bool gated = kKind == kMxGatedPair;
            const int m = gated ? 64 * p + (lane_p & 63) : 128 * p + lane_p;
            const bool up = gated && lane_p >= 64, live = m < A.outs;
            float bias = 0.f;
            if (A.bias != nullptr && live) bias = __uint_as_float(static_cast<uint32_t>(load_written(A.bias + m + (up ? A.outs : 0))) << 16);
            mt_wait(done + 8 * buf, buf_phase, &dead, 24);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem + buf * 256 + (static_cast<uint32_t>(quarter) << 21);
            for (int c = 0; c < cols; c += 32) {
                uint32_t r[32];
                asm volatile(
                    "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                    "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                    : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                      "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                      "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                    : "r"(from + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (c + 32 >= cols) {                                        // the accumulator is read: the issuer may have it back
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(free_ + 8 * buf);
                }
                if constexpr (!gated) {
                    if (live) {
                        uint16_t *to = A.out + static_cast<int64_t>(n0 + c) * A.outs + m;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c + i < cols) to[static_cast<int64_t>(i) * A.outs] = f32_to_bf16_rn(__uint_as_float(r[i]) + bias);
                    }
                } else {
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]) + bias;
                    if (A.pre != nullptr && live) {
                        float *to = A.pre + static_cast<int64_t>(n0 + c) * 2 * A.outs + m + (up ? A.outs : 0);
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c + i < cols) to[static_cast<int64_t>(i) * 2 * A.outs] = v[i];
                    }
                    // columns 0 .. 15 become the gate lanes', 16 .. 31 the up lanes': each hands the other half over
#pragma unroll
                    for (int i = 0; i < 16; i++) swap[((up ? 0 : 16) + i) * 64 + (lane_p & 63)] = up ? v[i] : v[16 + i];
                    asm volatile("bar.sync 2, 128;" ::: "memory");
                    if (live) {
                        const int i0 = up ? 16 : 0;
                        uint16_t *to = A.out + static_cast<int64_t>(n0 + c + i0) * A.outs + m;
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float other = swap[(i0 + i) * 64 + (lane_p & 63)];
                            const float g = up ? other : v[i], u = up ? v[16 + i] : other;
                            if (c + i0 + i < cols) to[static_cast<int64_t>(i) * A.outs] = f32_to_bf16_rn(mx_act(A.activation, g) * u);
                        }
                    }
                    asm volatile("bar.sync 2, 128;" ::: "memory");
                }
            }
            if ((buf ^= 1) == 0) buf_phase ^= 1u;
        }
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (dead)                                                                // copies and products under way land before the memory goes
        for (int i = 0; i < 10; i++) __nanosleep(100000);
    __syncthreads();
    if (warp == kMtIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace bhi
