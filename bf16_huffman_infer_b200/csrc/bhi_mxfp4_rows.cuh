// Products of 4-bit microscaled weights with few rows of X.
//
// y[r][m] = sum over blocks b of 2^(s[m][b] - 127) * sum over the block's k of code[m][k] x[r][k], and with kGated the rows g and u of a
// stacked weight at once, h = act(g) u: the 16 rows of a product are then the gates and ups of eight outputs, so that a lane has both.
//
// Bound by the bytes of the weight.  A warp takes one group of 128 columns of a step's MT tiles of 16 weight rows at a time.
// They come straight from global memory into registers, kDepth units ahead, and are multiplied by m16n8k16 products.
//
// Mostly the products are FP16 ones: the hardware's conversion makes two values of a code byte.  The sums of a block of 32 columns start at
// zero and its scale applies to them, in 32 bits, so codes need no scaling of their own.  X is brought to FP16 in shared memory: each row's 128
// values of a group to [2^14, 2^15) by a power of two that the sum gives back.  That is exact for every value down to 2^-31 of the largest in
// its 128, and down to 2^-28 the sums of blocks are multiples of 2^-22, whose products with any scale are whole steps of 2^-149.  Where one lies
// below (it may be all that counts: the weights of the large ones can be zero), X is brought once more and multiplied as it is, by the BF16 products
// of the next paragraph in a walk of its own.  (Looking for such values costs most where X is most of the work: 1024 x 4096, 1 row 4.65 against
// 4.52 us, 151936 x 4096, 8 rows 62 against 61, 38000 x 12288, 24 rows 118 against 115, gated 12288 x 4096, 16 rows 22.9 against 22.1; where there
// are some, 8 rows take 100 us.  A branch in every unit instead of the walk: 8 rows 66 us without any.)
// With X's power of two, up to 2^25 in four blocks, sums can overflow under a scale of 2^103 or more where the output does not: outputs that are
// not finite, of weight rows with large scales, are computed once more, one by one.  (Asking every unit for large scales took longer: 151936 x 4096, 1
// row 64 against 62 us.  Looking at the scales first: 151936 x 4096, 8 rows with a NaN in one 94 us, not 1255; 17 rows without 116 us, not 112.)
// Where there are more than eight rows to bring to FP16 and few steps to use them in, that takes longer than it saves: codes are expanded to
// BF16 with their scales, X is read as it is, and the products add up through all of K.
//
// The units of a CTA's steps, numbered through, are divided into one run for each warp: a step is one warp's but for those that the ends of
// runs cut.  The warp with a cut step's beginning adds the parts of the warps after it, in order (they had them at the beginning of their runs)
// and writes its outputs.  (With a step's groups dealt out to all warps, adding up fourteen parts a step took longer than the products
// from 16 rows on, whichever warps did it.)  Where X is too large for shared memory, K is walked in chunks: all steps of the CTA with one
// chunk's X, then with the next, the sums of each step kept in shared memory.
#pragma once

#include "bhi_mxfp4.cuh"

namespace bhi {

constexpr int kMxRowWarpsMax = 16;
constexpr uint32_t kMxRowsBelow = 28;             // powers of two between a group's largest value and the least that FP16 products serve

struct MxRowsArgs {
    MxWeight W;
    const uint16_t *X, *bias;
    uint16_t *Y;
    float *pre;                                   // gated, or null: [rows][2 * inter]
    int rows;
    int outs;                                     // M, or inter of a gated pair
    int activation;
    // the launch's plan
    int steps;                                    // plain: of MT tiles; gated: of 8 outputs
    int chunk_groups;                             // groups whose X lies in shared memory at a time
    uint32_t scale_off, part_off, sum_off;
};

__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

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

// A form of the kernel: MT tiles of weight rows by NT blocks of eight rows of X, kWarps warps, kDepth units in flight a warp, kPerSm CTAs an SM,
// FP16 or BF16 products.
template <int MT_, int NT_, int kWarps_, int kPerSm_, int kDepth_, bool kGated_, bool kHalf_ = true>
struct MxRowsForm {
    static constexpr int MT = MT_, NT = NT_, kWarps = kWarps_, kPerSm = kPerSm_, kDepth = kDepth_;
    static constexpr bool kGated = kGated_;
    static constexpr bool kHalf = kHalf_;                                    // FP16 products
    static constexpr int kThreads = 32 * kWarps_;
    static constexpr int kPlaces = kDepth_ + 1;                              // of a warp: the steps that end in a turn of kDepth units, and a part for another warp
    static_assert(kWarps <= kMxRowWarpsMax, "barriers");
    static constexpr int kPart = MT * NT * 32;                               // float4s of a warp's part of a step
    static_assert(!kGated || MT == 1, "a gated step is one tile");
    static __host__ __device__ uint32_t row_bytes(int chunk_groups) { return static_cast<uint32_t>(chunk_groups) * 256u + 64u; }     // rows 64 bytes apart in banks
};

// The larger and the smaller magnitude of each half; signs are left over (and a NaN is the larger).
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t min_abs_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Of eight BF16 values the largest magnitude (low half) and 65535 less the smallest (high half), as bits: both are found by maxima from here on.
__device__ __forceinline__ uint32_t mx_ends(const uint4 &v) {
    const uint32_t top = max_abs_bf16x2(max_abs_bf16x2(v.x, v.y), max_abs_bf16x2(v.z, v.w)) & 0x7FFF7FFFu;
    const uint32_t low = ~min_abs_bf16x2(min_abs_bf16x2(v.x, v.y), min_abs_bf16x2(v.z, v.w)) | 0x80008000u;
    return max_u16x2(__byte_perm(top, low, 0x5410), __byte_perm(top, low, 0x7632));
}
// Whether one of two BF16 values is neither zero nor as large as `from` (magnitudes as bits).
__device__ __forceinline__ bool mx_below(uint32_t pair, uint32_t from) {
    const uint32_t lo = pair & 0x7FFFu, hi = (pair >> 16) & 0x7FFFu;
    return (lo != 0u && lo < from) || (hi != 0u && hi < from);
}

// Whether weight row m has a scale of 2^65 or more (NaN scales aside): without one, a sum that is not finite is the output.
__device__ __forceinline__ bool mx_row_of_large_scales(const MxRowsArgs &A, int m) {
    const uint8_t *scales = A.W.scales + mx_scale_row(m, A.W.groups);
    uint32_t found = 0u;
    for (int g = 0; g < A.W.groups; g++) {
        const uint32_t s = load_stream4(scales + static_cast<int64_t>(g) * kMxTileScales);
        found |= s & (s << 1) & ~__vcmpeq4(s, 0xFFFFFFFFu);
    }
    return (found & 0x80808080u) != 0u;
}

// One output by itself: weight row m, row `col` of X, products in 32 bits.  Only if the weight row has large scales; otherwise what it `was`.
__device__ __forceinline__ float mx_one_output(const MxRowsArgs &A, int m, int col, float was) {
    if (!mx_row_of_large_scales(A, m)) return was;
    const uint8_t *codes = A.W.codes + mx_code_row(m, A.W.groups), *scales = A.W.scales + mx_scale_row(m, A.W.groups);
    const uint16_t *x = A.X + static_cast<int64_t>(col) * A.W.K;
    float sum = 0.f;
    for (int k = 0; k < A.W.K; k += 8) {
        const int g = k >> 7, j = (k >> 5) & 3, t = (k >> 3) & 3;
        float v[8];
        mx_word_to_f32(*reinterpret_cast<const uint32_t *>(codes + static_cast<int64_t>(g) * kMxTileCodes + t * 16 + j * 4),
                       mx_scale(scales[static_cast<int64_t>(g) * kMxTileScales + j]), v);
#pragma unroll
        for (int i = 0; i < 8; i++) sum = fmaf(v[i], __uint_as_float(static_cast<uint32_t>(load_written(x + k + i)) << 16), sum);
    }
    return sum;
}

template <class Form>
__global__ void __launch_bounds__(Form::kThreads, Form::kPerSm) mx_rows_kernel(const MxRowsArgs A) {
    constexpr int MT = Form::MT, NT = Form::NT, kDepth = Form::kDepth, kCols = 8 * NT;
    constexpr bool kGated = Form::kGated;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kMxRowWarpsMax + 1];
    __shared__ int not_fp16;                                                 // the last chunk (its number and one) with a value of X that FP16 does not hold
    __shared__ int dead;                                                     // a wait has run out: no other one waits any more
    constexpr int kWarps = Form::kWarps, threads = Form::kThreads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int my_steps = (A.steps - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const int chunks = (A.W.groups + A.chunk_groups - 1) / A.chunk_groups;
    const uint32_t base = smem_addr(smem);
    const uint32_t part_bar = smem_addr(&bars[0]), x_bar = part_bar + 8 * kMxRowWarpsMax;
    float4 *places = reinterpret_cast<float4 *>(smem + A.part_off), *sums = reinterpret_cast<float4 *>(smem + A.sum_off);

    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < kWarps; i++) mbar_init(part_bar + 8 * i, 1);
        mbar_init(x_bar, 1);
        mbar_fence_init();
        dead = 0;
        not_fp16 = 0;
    }
    __syncthreads();

    auto store = [&](int m, int col, float v, float u) {                     // u: of a gated pair
        if (m >= A.outs || col >= A.rows) return;
        const int64_t at = static_cast<int64_t>(col) * A.outs + m;
        if (A.bias != nullptr) {
            v += __uint_as_float(static_cast<uint32_t>(load_written(A.bias + m)) << 16);
            if constexpr (kGated) u += __uint_as_float(static_cast<uint32_t>(load_written(A.bias + A.outs + m)) << 16);
        }
        if constexpr (kGated) {
            A.Y[at] = f32_to_bf16_rn(mx_act(A.activation, v) * u);
            if (A.pre != nullptr) {
                A.pre[at + static_cast<int64_t>(col) * A.outs] = v;
                A.pre[at + static_cast<int64_t>(col + 1) * A.outs] = u;
            }
        } else {
            A.Y[at] = f32_to_bf16_rn(v);
        }
    };

    const uint32_t row_bytes = Form::row_bytes(A.chunk_groups);
    float *xscale = reinterpret_cast<float *>(smem + A.scale_off);
    uint32_t xat[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) xat[n] = static_cast<uint32_t>(min(8 * n + g, A.rows - 1)) * row_bytes + t * 16;

    // ---- the warp's run of units of a chunk, (step, group) pairs, kDepth ahead of their use ------------------------------------------------
    uint4 qa[kDepth][MT], qb[kDepth][MT];
    uint32_t sa[kDepth][MT], sb[kDepth][MT];
    // Rows a and b (eight on, or an output's up) of the step that is being requested, at the next group: 16-byte units of the codes of their
    // (tile, group) pairs, which are also bytes of the scales, and rows in their tiles.
    const uint8_t *codes = A.W.codes + t * 16, *scales = A.W.scales;
    constexpr int kRows = kGated ? 2 : MT;                                   // different (tile, group) pairs of a unit
    uint32_t at[kRows];
    int ra = g, rb = g + 8;
    int ask_step, ask_group, asked, run, units;
    auto run_of = [&](int w, int groups) { return static_cast<int>(static_cast<int64_t>(my_steps) * groups * w / kWarps); };      // where warp w's begins
    auto tiles_of = [&](int c0) {
        const int step = blockIdx.x + ask_step * gridDim.x;
        if constexpr (kGated) {                                              // past the last output (of the padded weight all the same): nobody reads the results
            const int ma = 8 * step + g, mb = A.outs + ma;
            at[0] = (static_cast<uint32_t>(ma >> 4) * A.W.groups + c0 + ask_group) * (kMxTileCodes / 16);
            at[1] = (static_cast<uint32_t>(mb >> 4) * A.W.groups + c0 + ask_group) * (kMxTileCodes / 16);
            ra = ma & 15;
            rb = mb & 15;
        } else {                                                             // past the last tile: the last one
#pragma unroll
            for (int q = 0; q < MT; q++)
                at[q] = (static_cast<uint32_t>(min(MT * step + q, (A.W.M - 1) >> 4)) * A.W.groups + c0 + ask_group) * (kMxTileCodes / 16);
        }
    };
    auto request = [&](int slot, int c0, int groups) {                       // past the last unit: the last one again, without effect
#pragma unroll
        for (int q = 0; q < MT; q++) {
            const uint32_t pa = at[q], pb = at[kGated ? 1 : q];
            const uint8_t *a = codes + static_cast<uint64_t>(pa) * 16 + ra * kMxRowCodes, *b = kGated ? codes + static_cast<uint64_t>(pb) * 16 + rb * kMxRowCodes : a + 8 * kMxRowCodes;
            qa[slot][q] = load_stream16(a);
            qb[slot][q] = load_stream16(b);
            sa[slot][q] = load_stream4(scales + pa + ra * 4);
            sb[slot][q] = load_stream4(scales + pb + rb * 4);
        }
        if (++asked < units) {
            if (++ask_group == groups) {
                ask_group = 0;
                ask_step++;
                tiles_of(c0);
            } else {
#pragma unroll
                for (int q = 0; q < kRows; q++) at[q] += kMxTileCodes / 16;
            }
        }
    };
    auto begin_chunk = [&](int c0, int groups) {
        run = run_of(warp, groups);
        units = run_of(warp + 1, groups) - run;
        ask_step = run / groups;
        ask_group = run - ask_step * groups;
        asked = 0;
        if (units > 0) {
            tiles_of(c0);
#pragma unroll
            for (int d = 0; d < kDepth; d++) request(d, c0, groups);
        }
    };
    begin_chunk(0, min(A.chunk_groups, A.W.groups));
    uint32_t x_phase = 0u;
    for (int c = 0; c < chunks; c++) {
        const int c0 = c * A.chunk_groups, groups = min(A.chunk_groups, A.W.groups - c0);

        // X: rows as they are by the copy engine, then to FP16 fragments in place: chunk (group, block, quarter) is eight values, in the
        // order of a word's nibbles
        const int x_bytes = 2 * min(A.W.K - c0 * kMxGroup, groups * kMxGroup);       // of a row
        if (c > 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            begin_chunk(c0, groups);
            __syncthreads();                                                      // nobody reads the last chunk's X any more
        }
        auto bring_x = [&]() {
            if (warp == 0) {
                if (lane == 0) mbar_expect_tx(x_bar, static_cast<uint32_t>(x_bytes * A.rows));
                __syncwarp();
                if (lane < A.rows) bulk_copy_g2s(base + lane * row_bytes, A.X + static_cast<int64_t>(lane) * A.W.K + c0 * kMxGroup, x_bytes, x_bar);
            }
            mx_wait(x_bar, x_phase, &dead, 11);
            x_phase ^= 1u;
        };
        auto pad_x = [&]() {                                                 // past the last column: zeros
            const int pad = groups * 256 - x_bytes;
            for (int i = tid * 16; i < A.rows * pad; i += threads * 16) *reinterpret_cast<uint4 *>(smem + i / pad * row_bytes + x_bytes + i % pad) = make_uint4(0u, 0u, 0u, 0u);
        };
        if (c == 0 && warp == 0) pdl_wait();
        bring_x();
        bool fp16 = Form::kHalf;                                             // FP16 products, here and now
        if constexpr (Form::kHalf) {
            // to FP16 in place: chunk (group, block, quarter) is eight values, in the order of a word's nibbles; half a warp takes a group of a
            // row, four of them at once
            constexpr int kAtOnce = 4;
            const int teams = threads / 16, ch = lane & 15, jobs = groups * A.rows, on = teams / A.rows, more = teams - on * A.rows;
            const uint32_t half = 0xFFFFu << (lane & 16);
            int xg = (tid >> 4) / A.rows, xr = (tid >> 4) - xg * A.rows;
            bool far = false;                                                // a value that FP16 does not hold
            for (int job0 = tid >> 4; job0 < jobs; job0 += teams * kAtOnce) {
                uint32_t w[kAtOnce][4], ends[kAtOnce], at_x[kAtOnce], at_s[kAtOnce];
#pragma unroll
                for (int q = 0; q < kAtOnce; q++) {
                    at_x[q] = xr * row_bytes + xg * 256 + ch * 16;
                    at_s[q] = xg * kCols + xr;
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (job0 + q * teams < jobs && xg * 256 + ch * 16 < x_bytes) v = *reinterpret_cast<const uint4 *>(smem + at_x[q]);
                    w[q][0] = v.x, w[q][1] = v.y, w[q][2] = v.z, w[q][3] = v.w;
                    ends[q] = mx_ends(v);                                    // (an infinity or NaN makes the whole row one, whatever becomes of its other values)
                    xg += on;
                    xr += more;
                    if (xr >= A.rows) xr -= A.rows, xg++;
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                    for (int q = 0; q < kAtOnce; q++) ends[q] = max_u16x2(ends[q], __shfl_xor_sync(half, ends[q], o));
#pragma unroll
                for (int q = 0; q < kAtOnce; q++) {
                    if (job0 + q * teams >= jobs) break;
                    const uint32_t top = ends[q] & 0xFF80u;                  // without its mantissa
                    const uint32_t up = min(268u - (top >> 7), 253u);        // exponent field of 2^(14 - floor(log2 top))
                    // the smallest is too far below: a zero, or (next to an infinity or NaN that does not matter) a value that FP16 products do not serve
                    if ((ends[q] >> 16) + top > 0xFFFFu + (kMxRowsBelow << 7) && top < 0x7F80u)
                        for (int i = 0; i < 4; i++) far |= mx_below(w[q][i], top - (kMxRowsBelow << 7));
                    const float scale = __uint_as_float(up << 23);
                    uint32_t h[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        // (e0, e2) (e4, e6) (e1, e3) (e5, e7): element e is half e & 1 of word e >> 1
                        const uint32_t a = w[q][(j & 1) * 2], b = w[q][(j & 1) * 2 + 1];
                        const float lo = (j >> 1 ? bf16hi_to_f32(a) : bf16lo_to_f32(a)) * scale, hi = (j >> 1 ? bf16hi_to_f32(b) : bf16lo_to_f32(b)) * scale;
                        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[j]) : "f"(hi), "f"(lo));
                    }
                    *reinterpret_cast<uint4 *>(smem + at_x[q]) = make_uint4(h[0], h[1], h[2], h[3]);
                    if (ch == 0) xscale[at_s[q]] = __uint_as_float((254u - up) << 23);
                }
            }
            if (far) not_fp16 = c + 1;
            __syncthreads();
            fp16 = not_fp16 != c + 1;
            if (!fp16) {                                                     // X as it is
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncthreads();
                bring_x();
                pad_x();
                __syncthreads();
            }
        } else {
            pad_x();
            __syncthreads();
        }

        float acc[MT][NT][4];
#pragma unroll
        for (int q = 0; q < MT; q++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) acc[q][n][k] = 0.f;
        const int run_step = run / groups;                                   // the local step in which the run begins
        int i = run_step, gr = run - i * groups, first = i;                  // step and group of the unit at hand; the first step not dealt with
        const bool begun = gr == 0;                                          // the run begins with its step
        auto multiply_f16 = [&](int d) {
            uint32_t pa[MT][2], pb[MT][2];                                   // the blocks' scales in BF16
#pragma unroll
            for (int q = 0; q < MT; q++) {
                mx_scales_bf16(sa[d][q], pa[q]);
                mx_scales_bf16(sb[d][q], pb[q]);
            }
            float cg[MT][NT][4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint4 x[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) x[n] = *reinterpret_cast<const uint4 *>(smem + xat[n] + gr * 256 + j * 64);
#pragma unroll
                for (int q = 0; q < MT; q++) {
                    const uint4 &wa = qa[d][q], &wb = qb[d][q];
                    uint32_t ha[4], hb[4];
                    mx_word_to_f16(j == 0 ? wa.x : j == 1 ? wa.y : j == 2 ? wa.z : wa.w, ha);
                    mx_word_to_f16(j == 0 ? wb.x : j == 1 ? wb.y : j == 2 ? wb.z : wb.w, hb);
                    const float fa = j & 1 ? bf16hi_to_f32(pa[q][j >> 1]) : bf16lo_to_f32(pa[q][j >> 1]), fb = j & 1 ? bf16hi_to_f32(pb[q][j >> 1]) : bf16lo_to_f32(pb[q][j >> 1]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float e[4];
                        mma_f16_first(e, ha[0], hb[0], ha[1], hb[1], x[n].x, x[n].y);
                        mma_f16(e, ha[2], hb[2], ha[3], hb[3], x[n].z, x[n].w);
#pragma unroll
                        for (int k = 0; k < 4; k++) cg[q][n][k] = j == 0 ? e[k] * (k < 2 ? fa : fb) : fmaf(e[k], k < 2 ? fa : fb, cg[q][n][k]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float2 xs = *reinterpret_cast<const float2 *>(xscale + gr * kCols + 8 * n + 2 * t);
#pragma unroll
                for (int q = 0; q < MT; q++)
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[q][n][k] = fmaf(cg[q][n][k], k & 1 ? xs.y : xs.x, acc[q][n][k]);
            }
        };
        auto multiply_bf16 = [&](int d, auto large) {
            constexpr bool kLarge = decltype(large)::value;
            uint32_t fa[MT][4], fb[MT][4];
#pragma unroll
            for (int q = 0; q < MT; q++) {
                mx_factors<kLarge>(sa[d][q], fa[q]);
                mx_factors<kLarge>(sb[d][q], fb[q]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint4 x[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) x[n] = *reinterpret_cast<const uint4 *>(smem + xat[n] + gr * 256 + j * 64);
#pragma unroll
                for (int q = 0; q < MT; q++) {
                    const uint4 a = mx_word_to_bf16<kLarge>(word_of(qa[d][q], j), fa[q][j]), b = mx_word_to_bf16<kLarge>(word_of(qb[d][q], j), fb[q][j]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma_bf16_16x8x16(acc[q][n], a.x, b.x, a.y, b.y, x[n].x, x[n].y);
                        mma_bf16_16x8x16(acc[q][n], a.z, b.z, a.w, b.w, x[n].z, x[n].w);
                    }
                }
            }
        };
        auto multiply = [&](int d, auto as_half) {
            if constexpr (decltype(as_half)::value) {
                multiply_f16(d);
            } else {
                uint32_t any = 0u;
#pragma unroll
                for (int q = 0; q < MT; q++) any |= sa[d][q] | sb[d][q];
                if (Form::kHalf || __any_sync(0xFFFFFFFFu, (any & 0x80808080u) != 0u)) multiply_bf16(d, std::true_type{});
                else multiply_bf16(d, std::false_type{});
            }
            gr++;
        };
        // the sums so far to one of this warp's places, and to zero
        auto put = [&](int place) {
            float4 *dst = places + (warp * Form::kPlaces + place) * Form::kPart + lane;
#pragma unroll
            for (int q = 0; q < MT; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    dst[(q * NT + n) * 32] = make_float4(acc[q][n][0], acc[q][n][1], acc[q][n][2], acc[q][n][3]);
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[q][n][k] = 0.f;
                }
        };
        // Every warp once a chunk: its part of a step that another one began, if it has any, is in its last place.
        auto hand_over = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(part_bar + 8 * warp);
        };
        // the outputs of a step from one of this warp's places and the parts of the warps up to `others`
        auto finish = [&](int local, int place, int others) {
            const int step = blockIdx.x + local * gridDim.x;
            const float4 *own = places + (warp * Form::kPlaces + place) * Form::kPart;
            if (lane < others - warp) mx_wait(part_bar + 8 * (warp + 1 + lane), c & 1, &dead, 12);
            __syncwarp();
            const bool few = my_steps * groups < kWarps;                     // some runs are empty
            constexpr int kItems = MT * NT, kUnroll = kItems == 1 ? 4 : 1;   // (more code costs more than it hides)
#pragma unroll 1
            for (int item = 0; item < kItems; item++) {
                const int at_v = item * 32 + lane, n = item % NT;
                float4 v = own[at_v];
#pragma unroll(kUnroll)
                for (int w = warp + 1; w <= others; w++) {
                    if (few && run_of(w, groups) == run_of(w + 1, groups)) continue;
                    const float4 p = places[(w * Form::kPlaces + kDepth) * Form::kPart + at_v];
                    v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
                }
                float4 *keep = sums + local * Form::kPart + at_v;
                if (c > 0) {
                    const float4 p = *keep;
                    v.x += p.x, v.y += p.y, v.z += p.z, v.w += p.w;
                }
                if (c + 1 < chunks) {
                    *keep = v;
                    continue;
                }
                const int col = 8 * n + 2 * t;
                if constexpr (Form::kHalf) {
                    const bool even = !(isfinite(v.x) && isfinite(v.z)), odd = !(isfinite(v.y) && isfinite(v.w));
                    if ((even && col < A.rows) || (odd && col + 1 < A.rows)) {
                        const int ma = kGated ? 8 * step + g : 16 * (MT * step + item / NT) + g, mb = kGated ? A.outs + ma : ma + 8;
#pragma unroll 1
                        for (int k = 0; k < 4; k++) {
                            const int m = k < 2 ? ma : mb;
                            if (!(k & 1 ? odd : even) || col + (k & 1) >= A.rows || (kGated ? ma : m) >= A.outs) continue;
                            const float one = mx_one_output(A, m, col + (k & 1), k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w);
                            if (k == 0) v.x = one;
                            if (k == 1) v.y = one;
                            if (k == 2) v.z = one;
                            if (k == 3) v.w = one;
                        }
                    }
                }
                if constexpr (kGated) {
                    store(8 * step + g, col, v.x, v.z);
                    store(8 * step + g, col + 1, v.y, v.w);
                } else {
                    const int m = 16 * (MT * step + item / NT) + g;
                    store(m, col, v.x, 0.f);
                    store(m, col + 1, v.y, 0.f);
                    store(m + 8, col, v.z, 0.f);
                    store(m + 8, col + 1, v.w, 0.f);
                }
            }
            __syncwarp();                                                    // every lane has read the place
        };
        bool handed = false;
        auto end_of_step = [&]() {
            gr = 0;
            put(i == run_step && !begun ? kDepth : i - first);
            i++;
        };
        auto finish_steps = [&]() {                                          // those that ended since the last time
            __syncwarp();
            for (int place = 0; first < i; first++, place++) {
                if (first == run_step && !begun) hand_over(), handed = true;
                else finish(first, place, warp);
            }
        };
        auto walk = [&](auto as_half) {
            int u = 0;
            for (; u + kDepth <= units; u += kDepth) {
#pragma unroll
                for (int d = 0; d < kDepth; d++) {
                    multiply(d, as_half);
                    request(d, c0, groups);
                    if (gr == groups) end_of_step();
                }
                if (first < i) finish_steps();
            }
#pragma unroll
            for (int d = 0; d < kDepth; d++) {
                if (u + d < units) {
                    multiply(d, as_half);
                    if (gr == groups) end_of_step();
                }
            }
            if (first < i) finish_steps();
        };
        if constexpr (Form::kHalf) {
            if (fp16) walk(std::true_type{});
            else walk(std::false_type{});
        } else {
            walk(std::false_type{});
        }
        int others = warp;
        const bool cut = gr != 0 && units > 0, mine = i > run_step || begun;       // the run ends inside a step; which this warp began
        if (cut) put(mine ? 0 : kDepth);
        if (!handed) hand_over();
        if (cut && mine) {
            while (others + 1 < kWarps && run_of(others + 1, groups) < (i + 1) * groups) others++;
            finish(i, 0, others);
        }
    }
}

}  // namespace bhi
