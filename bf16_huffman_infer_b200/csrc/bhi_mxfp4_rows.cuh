// Products of 4-bit microscaled weights with few rows of X.
//
// y[r][m] = sum over blocks b of 2^(s[m][b] - 127) * sum over the block's k of code[m][k] x[r][k], and with kGated the rows g and u of a
// stacked weight at once, h = act(g) u.
//
// Bound by the bytes of the weight.  A warp takes 16 rows and one group of 128 columns at a time, straight from global memory into
// registers (two 16-byte loads a lane, kDepth such units in flight), turns the codes into FP16 by the hardware's conversion and
// multiplies blocks of 32 columns by m16n8k16 products whose sums start at zero: a block's scale applies to its sum, in 32 bits, so
// codes need no scaling of their own.  X is FP16 there: each row's 128 values of a group are brought to [2^14, 2^15) by a power of two
// that the sum gives back.  That is exact for every value down to 2^-32 of the largest in its 128; below, the error is
// under 2^-40 of that largest one, far less than a 32-bit sum with it loses.
//
// The eight warps of a CTA (and the CTAs of a cluster, where K x rows is too much shared memory for one) divide the groups, each
// adding up its own; the parts of kBatch steps are put together in shared memory at a time, in a fixed order.
#pragma once

#include "bhi_mxfp4.cuh"

namespace bhi {

constexpr int kMxRowThreads = 256;
constexpr int kMxRowWarps = 8;
constexpr int kMxBatch = 4;                       // steps whose parts are put together at a time
constexpr int kMxClusterMax = 8;

struct MxRowsArgs {
    MxWeight W;
    const uint16_t *X, *bias;
    uint16_t *Y;
    float *pre;                                   // gated, or null: [rows][2 * inter]
    int rows;
    int outs;                                     // M, or inter of a gated pair
    int steps;                                    // 16 outputs a step (8 gated ones)
    int part_groups;                              // groups of a CTA of the cluster
    int activation;
};

__device__ __forceinline__ uint4 load_stream16(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_stream4(const uint8_t *p) {
    uint32_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load_written16(const uint16_t *p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_load(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// shared memory: X fragments, their scales, the warps' parts, the CTA's parts (two batches, only of a cluster)
template <int NT>
struct MxRowsPlan {
    static constexpr int kCols = 8 * NT;
    static constexpr int kParts = kMxBatch * kMxRowWarps * NT * 128;         // floats
    static constexpr int kSums = kMxBatch * 16 * kCols;                      // floats of a batch
    static __host__ __device__ uint32_t row_bytes(int part_groups) { return static_cast<uint32_t>(part_groups) * 256u + 64u; }     // rows 64 bytes apart in banks
    static __host__ __device__ uint32_t scale_off(int rows, int part_groups) { return static_cast<uint32_t>(rows) * row_bytes(part_groups); }
    static __host__ __device__ uint32_t part_off(int rows, int part_groups) { return scale_off(rows, part_groups) + static_cast<uint32_t>(part_groups) * kCols * 4u; }
    static __host__ __device__ uint32_t total(int rows, int part_groups, int cluster) {
        return part_off(rows, part_groups) + kParts * 4u + (cluster > 1 ? 2u * kSums * 4u : 0u);
    }
};

template <int NT, int kDepth, bool kGated>
__global__ void __launch_bounds__(kMxRowThreads, 2) mx_rows_kernel(const MxRowsArgs A) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using Plan = MxRowsPlan<NT>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int size = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
    const int first_step = blockIdx.x / size, stride = gridDim.x / size;
    const int group0 = rank * A.part_groups;
    const int groups = max(0, min(A.W.groups - group0, A.part_groups));      // of this CTA
    const int mine = (groups - warp + kMxRowWarps - 1) / kMxRowWarps;        // of this warp: warp, warp + 8, ...
    const int my_steps = first_step < A.steps ? (A.steps - first_step + stride - 1) / stride : 0;

    pdl_launch_dependents();

    // ---- the stream of units: (step, group) pairs of this warp, kDepth ahead ---------------------------------------------
    uint4 qa[kDepth], qb[kDepth];
    uint32_t sa[kDepth], sb[kDepth];
    const uint8_t *ca, *cb, *ea, *eb;                                        // rows of the step that is being requested
    auto rows_of = [&](int step) {
        int ma, mb;
        if constexpr (kGated) {
            ma = min(8 * step + g, A.outs - 1);                              // past the last one: nobody reads the result
            mb = ma + A.outs;
        } else {
            ma = 16 * step + g;                                              // rows up to the end of the tile exist
            mb = ma + 8;
        }
        const int64_t at = group0 + warp;
        ca = A.W.codes + mx_code_row(ma, A.W.groups) + at * kMxTileCodes + t * 16;
        cb = A.W.codes + mx_code_row(mb, A.W.groups) + at * kMxTileCodes + t * 16;
        ea = A.W.scales + mx_scale_row(ma, A.W.groups) + at * kMxTileScales;
        eb = A.W.scales + mx_scale_row(mb, A.W.groups) + at * kMxTileScales;
    };
    const int total = mine > 0 ? my_steps * mine : 0;
    int asked = 0, ask_group = 0, ask_step = first_step;
    if (total > 0) rows_of(ask_step);
    auto request = [&](int slot) {
        if (asked < total) {
            qa[slot] = load_stream16(ca);
            qb[slot] = load_stream16(cb);
            sa[slot] = load_stream4(ea);
            sb[slot] = load_stream4(eb);
            asked++;
            ca += kMxRowWarps * kMxTileCodes;
            cb += kMxRowWarps * kMxTileCodes;
            ea += kMxRowWarps * kMxTileScales;
            eb += kMxRowWarps * kMxTileScales;
            if (++ask_group == mine) {
                ask_group = 0;
                ask_step += stride;
                if (asked < total) rows_of(ask_step);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < kDepth; d++) request(d);

    // ---- X to FP16 fragments: chunk (group, block, quarter) of a row is eight values, in the order of a word's nibbles --------
    pdl_wait();
    const uint32_t row_bytes = Plan::row_bytes(A.part_groups);
    float *xscale = reinterpret_cast<float *>(smem + Plan::scale_off(A.rows, A.part_groups));
    for (int i = tid >> 4; i < A.rows * groups; i += kMxRowThreads / 16) {
        const int r = i / groups, gr = i % groups, c = lane & 15;
        const int k = (group0 + gr) * kMxGroup + c * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (k < A.W.K) v = load_written16(A.X + static_cast<int64_t>(r) * A.W.K + k);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t top = 0u;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t lo = w[j] & 0x7FFFu, hi = (w[j] >> 16) & 0x7FFFu;
            top = max(top, lo < 0x7F80u ? lo : 0u);                          // infinities and NaNs keep themselves whatever the scale
            top = max(top, hi < 0x7F80u ? hi : 0u);
        }
        const uint32_t half = 0xFFFFu << (lane & 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(half, top, o));
        const uint32_t up = min(268u - (top >> 7), 253u);                    // exponent field of 2^(14 - floor(log2 top))
        const float scale = __uint_as_float(up << 23);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            f[2 * j] = bf16lo_to_f32(w[j]) * scale;
            f[2 * j + 1] = bf16hi_to_f32(w[j]) * scale;
        }
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // (e0, e2) (e4, e6) (e1, e3) (e5, e7)
            const int e = (j & 1) * 4 + (j >> 1);
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[j]) : "f"(f[e + 2]), "f"(f[e]));
        }
        *reinterpret_cast<uint4 *>(smem + r * row_bytes + gr * 256 + c * 16) = make_uint4(h[0], h[1], h[2], h[3]);
        if (c == 0) xscale[gr * Plan::kCols + r] = __uint_as_float((254u - up) << 23);
    }
    __syncthreads();

    // ---- the products -------------------------------------------------------------------------------------------------------
    float *parts = reinterpret_cast<float *>(smem + Plan::part_off(A.rows, A.part_groups));
    float *sums = parts + Plan::kParts;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[n][c] = 0.f;
    uint32_t xat[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) xat[n] = static_cast<uint32_t>(min(8 * n + g, A.rows - 1)) * row_bytes + t * 16;

    auto multiply = [&](const uint4 &wa, const uint4 &wb, uint32_t ka, uint32_t kb, int gr) {
        const uint32_t va[4] = {wa.x, wa.y, wa.z, wa.w}, vb[4] = {wb.x, wb.y, wb.z, wb.w};
        float cg[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) cg[n][c] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t ha[4], hb[4];
            mx_word_to_f16(va[j], ha);
            mx_word_to_f16(vb[j], hb);
            // byte j of the scale words to the exponent field; the smallest scale, 2^-127, counts as zero here
            const float fa = __uint_as_float(j < 3 ? (ka << (23 - 8 * j)) & 0x7F800000u : (ka >> 1) & 0x7F800000u);
            const float fb = __uint_as_float(j < 3 ? (kb << (23 - 8 * j)) & 0x7F800000u : (kb >> 1) & 0x7F800000u);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(smem + xat[n] + gr * 256 + j * 64);
                float c[4];
                mma_f16_first(c, ha[0], hb[0], ha[1], hb[1], x.x, x.y);
                mma_f16(c, ha[2], hb[2], ha[3], hb[3], x.z, x.w);
                cg[n][0] = fmaf(c[0], fa, cg[n][0]);
                cg[n][1] = fmaf(c[1], fa, cg[n][1]);
                cg[n][2] = fmaf(c[2], fb, cg[n][2]);
                cg[n][3] = fmaf(c[3], fb, cg[n][3]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float2 xs = *reinterpret_cast<const float2 *>(xscale + gr * Plan::kCols + 8 * n + 2 * t);
            acc[n][0] = fmaf(cg[n][0], xs.x, acc[n][0]);
            acc[n][1] = fmaf(cg[n][1], xs.y, acc[n][1]);
            acc[n][2] = fmaf(cg[n][2], xs.x, acc[n][2]);
            acc[n][3] = fmaf(cg[n][3], xs.y, acc[n][3]);
        }
    };

    // an output of a batch: value (row in step, column of X) as the sum of the warps' parts
    auto part_sum = [&](int p, int row, int col) {
        const float *src = parts + ((p * kMxRowWarps * NT + (col >> 3)) * 32 + (row & 7) * 4 + ((col & 7) >> 1)) * 4 + (row >> 3) * 2 + (col & 1);
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kMxRowWarps; w++) s += src[w * NT * 128];
        return s;
    };
    auto finish = [&](int step0, int steps) {                                // `steps` steps from step0 on are in `parts`
        __syncthreads();
        const uint32_t sums_at = smem_addr(sums) + ((step0 / kMxBatch) & 1) * Plan::kSums * 4u;
        if (size > 1) {
            float *mine_sums = sums + ((step0 / kMxBatch) & 1) * Plan::kSums;
            for (int i = tid; i < steps * 16 * A.rows; i += kMxRowThreads) {
                const int row = i & 15, p = (i >> 4) % steps, col = (i >> 4) / steps;
                mine_sums[(p * Plan::kCols + col) * 16 + row] = part_sum(p, row, col);
            }
            cluster_sync();
        }
        auto value = [&](int p, int row, int col) {
            if (size == 1) return part_sum(p, row, col);
            float s = 0.f;
            for (int q = 0; q < size; q++) s += cluster_load(sums_at + ((p * Plan::kCols + col) * 16 + row) * 4, q);
            return s;
        };
        constexpr int kPer = kGated ? 8 : 16;
        // row fastest: neighbouring threads write neighbouring outputs
        for (int i = tid + rank * kMxRowThreads; i < steps * kPer * A.rows; i += kMxRowThreads * size) {
            const int row = i % kPer, p = i / kPer % steps, col = i / (kPer * steps);
            const int m = (first_step + (step0 + p) * stride) * kPer + row;
            if (m >= A.outs) continue;
            if constexpr (kGated) {
                float gv = value(p, row, col), uv = value(p, row + 8, col);
                if (A.bias != nullptr) {
                    gv += __uint_as_float(static_cast<uint32_t>(load_written(A.bias + m)) << 16);
                    uv += __uint_as_float(static_cast<uint32_t>(load_written(A.bias + A.outs + m)) << 16);
                }
                A.Y[static_cast<int64_t>(col) * A.outs + m] = f32_to_bf16_rn(mx_act(A.activation, gv) * uv);
                if (A.pre != nullptr) {
                    A.pre[static_cast<int64_t>(col) * 2 * A.outs + m] = gv;
                    A.pre[static_cast<int64_t>(col) * 2 * A.outs + A.outs + m] = uv;
                }
            } else {
                float v = value(p, row, col);
                if (A.bias != nullptr) v += __uint_as_float(static_cast<uint32_t>(load_written(A.bias + m)) << 16);
                A.Y[static_cast<int64_t>(col) * A.outs + m] = f32_to_bf16_rn(v);
            }
        }
        __syncthreads();
    };

    int step = 0, group = 0, gr = warp;
    auto end_of_step = [&]() {                                               // this warp's part of a step is complete
        float *dst = parts + (((step % kMxBatch) * kMxRowWarps + warp) * NT * 32 + lane) * 4;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            *reinterpret_cast<float4 *>(dst + n * 128) = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
#pragma unroll
            for (int c = 0; c < 4; c++) acc[n][c] = 0.f;
        }
        step++;
        if (step % kMxBatch == 0) finish(step - kMxBatch, kMxBatch);
    };
    if (total == 0) {
        while (step < my_steps) end_of_step();                               // a warp without groups still adds its zeros
    } else {
        for (int u = 0; u < total; u += kDepth) {
#pragma unroll
            for (int d = 0; d < kDepth; d++) {
                if (u + d < total) {
                    multiply(qa[d], qb[d], sa[d], sb[d], gr);
                    request(d);
                    gr += kMxRowWarps;
                    if (++group == mine) {
                        group = 0;
                        gr = warp;
                        end_of_step();
                    }
                }
            }
        }
    }
    if (step % kMxBatch != 0) finish(step - step % kMxBatch, step % kMxBatch);
    if (size > 1) cluster_sync();                                            // nobody reads this CTA's sums any more
}

}  // namespace bhi
