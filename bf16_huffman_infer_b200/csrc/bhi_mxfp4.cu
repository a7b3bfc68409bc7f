// 4-bit microscaled weights: quantisation, the dense matrix, products.
#include "bhi_mxfp4.cuh"

namespace bhi {

// ---- quantisation ----------------------------------------------------------------------------------------------------
// Per block of 32: e = floor(log2 max|v|) - 2 (the largest code is 6 = 1.5 * 2^2), not below -127; codes are v / 2^e rounded to the
// nearest, ties to the even code, saturated at 6.  A power of two divides exactly, subnormal values included, and the
// hardware's conversion rounds and saturates so: every code is the format's own.  A block with an infinity or a NaN is NaN.
//
// A thread makes a word (8 values) of each of kMxQuantRows rows at once, the four threads of a block share its maximum; a warp reads
// 256 values of a row in one piece and writes them as two of 64 bytes, four rows side by side.  Bound by memory: read once, written once.
template <class T>
__device__ __forceinline__ void mx_load8(const T *p, uint32_t (&bits)[8]);
template <>
__device__ __forceinline__ void mx_load8<__nv_bfloat16>(const __nv_bfloat16 *p, uint32_t (&bits)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bits[2 * i] = w[i] << 16;
        bits[2 * i + 1] = w[i] & 0xFFFF0000u;
    }
}
template <>
__device__ __forceinline__ void mx_load8<__half>(const __half *p, uint32_t (&bits)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bits[2 * i] = __float_as_uint(f16lo_to_f32(w[i]));
        bits[2 * i + 1] = __float_as_uint(f16hi_to_f32(w[i]));
    }
}
template <>
__device__ __forceinline__ void mx_load8<float>(const float *p, uint32_t (&bits)[8]) {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p)), b = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; i++) bits[i] = w[i];
}

constexpr int kMxQuantThreads = 512;                                     // at most
constexpr int kMxQuantRows = 4;

template <class T>
__global__ void __launch_bounds__(kMxQuantThreads) mx_quantize_kernel(const T *W, int M, int K, int groups, uint8_t *codes, uint8_t *scales) {
    const int at = blockIdx.x * blockDim.x + threadIdx.x;                // word of a row
    const bool in_row = at < groups * 16;
    const int g = at >> 4, j = (at >> 2) & 3, t = at & 3;
    const int tiles16 = (M + 15) / 16 * 16;
    for (int m0 = blockIdx.y * kMxQuantRows; m0 < tiles16; m0 += gridDim.y * kMxQuantRows) {       // 16 is a multiple of kMxQuantRows
        uint32_t v[kMxQuantRows][8];
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[r][i] = 0u;
            if (m0 + r < M && at * 8 < K) mx_load8(W + static_cast<int64_t>(m0 + r) * K + at * 8, v[r]);
        }
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) {
            uint32_t top = 0u;
#pragma unroll
            for (int i = 0; i < 8; i++) top = max(top, v[r][i] & 0x7FFFFFFFu);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t field = top >> 23;                             // floor(log2 top) + 127 of a normal value
            const bool nan = field == 255u;
            const uint32_t byte = nan ? 255u : field > 2u ? field - 2u : 0u;
            const float inv = __uint_as_float((254u - byte) << 23);       // 2^(127 - byte); not used for a NaN
            uint32_t word = 0u;
            if (!nan) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] = __uint_as_float(v[r][i]) * inv;
                // bytes: (e0, e2) (e4, e6) (e1, e3) (e5, e7), the first in the low half
                asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
                    "cvt.rn.satfinite.e2m1x2.f32 b0, %3, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %7, %5;\n\t"
                    "cvt.rn.satfinite.e2m1x2.f32 b2, %4, %2;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %6;\n\t"
                    "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
                    : "=r"(word) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
            }
            if (in_row) {
                const int64_t row = mx_code_row(m0 + r, groups);
                *reinterpret_cast<uint32_t *>(codes + row + static_cast<int64_t>(g) * kMxTileCodes + t * 16 + j * 4) = word;
                if (t == 0) scales[mx_scale_row(m0 + r, groups) + static_cast<int64_t>(g) * kMxTileScales + j] = static_cast<uint8_t>(byte);
            }
        }
    }
}

// ---- from the plain order ----------------------------------------------------------------------------------------------
// Two codes a byte along a row, the even element in the low half, and a scale byte a block, to the order of the kernels; threads as above.
// Scales of 2^126 and 2^127, under which some codes leave the range of BF16 and of 32-bit floats, are not stored, so that whatever multiplies by
// codes and scales apart agrees with whatever multiplies by values: a block without such codes is the same values under 2^125, one with any
// has infinities and is NaN, as in quantisation.

// The codes of a word of a block under 2^(125 + up) as those under 2^125; those that have none make `beyond` true.
__device__ __forceinline__ uint32_t mx_codes_under_125(uint32_t word, uint32_t up, bool &beyond) {
    // of 0, 0.5, 1, 1.5, 2, 3, 4, 6 the codes of twice and four times the value
    const uint32_t codes = up == 1u ? 0x00765420u : 0x00007640u, most = up == 1u ? 5u : 3u;
    uint32_t out = word & 0x88888888u;
    for (int i = 0; i < 32; i += 4) {
        const uint32_t magnitude = (word >> i) & 7u;
        beyond |= magnitude > most;
        out |= ((codes >> (4 * magnitude)) & 7u) << i;
    }
    return out;
}
__global__ void __launch_bounds__(kMxQuantThreads) mx_layout_kernel(const uint8_t *packed, const uint8_t *packed_scales, int M, int K, int groups, uint8_t *codes, uint8_t *scales) {
    const int at = blockIdx.x * blockDim.x + threadIdx.x;                // word of a row
    const bool in_row = at < groups * 16;
    const int g = at >> 4, j = (at >> 2) & 3, t = at & 3;
    const int tiles16 = (M + 15) / 16 * 16;
    for (int m0 = blockIdx.y * kMxQuantRows; m0 < tiles16; m0 += gridDim.y * kMxQuantRows) {
        uint32_t word[kMxQuantRows], byte[kMxQuantRows];
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) {
            word[r] = byte[r] = 0u;
            if (m0 + r < M && at * 8 < K) {
                word[r] = __ldg(reinterpret_cast<const uint32_t *>(packed + static_cast<int64_t>(m0 + r) * (K / 2)) + at);
                byte[r] = __ldg(packed_scales + static_cast<int64_t>(m0 + r) * (K / 32) + (at >> 2));
            }
        }
        bool high = false;
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) high |= byte[r] == 253u || byte[r] == 254u;
        if (__any_sync(0xFFFFFFFFu, high)) {
#pragma unroll
            for (int r = 0; r < kMxQuantRows; r++) {
                bool beyond = false;
                if (byte[r] == 253u || byte[r] == 254u) word[r] = mx_codes_under_125(word[r], byte[r] - 252u, beyond), byte[r] = 252u;
                uint32_t nan = beyond ? 1u : 0u;                             // anywhere in the block: its four threads
                nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 1);
                nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 2);
                if (nan) byte[r] = 255u;
            }
        }
        if (!in_row) continue;
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) {
            uint32_t even = word[r] & 0x0F0F0F0Fu, odd = (word[r] >> 4) & 0x0F0F0F0Fu;      // a nibble a byte: side by side, in two steps
            even = (even | even >> 4) & 0x00FF00FFu, odd = (odd | odd >> 4) & 0x00FF00FFu;
            even = (even | even >> 8) & 0xFFFFu, odd = (odd | odd >> 8) & 0xFFFFu;
            const int64_t row = mx_code_row(m0 + r, groups);
            *reinterpret_cast<uint32_t *>(codes + row + static_cast<int64_t>(g) * kMxTileCodes + t * 16 + j * 4) = byte[r] == 255u ? 0u : even | odd << 16;
            if (t == 0) scales[mx_scale_row(m0 + r, groups) + static_cast<int64_t>(g) * kMxTileScales + j] = static_cast<uint8_t>(byte[r]);
        }
    }
}

// ---- the dense matrix ------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kMxQuantThreads) mx_dense_kernel(MxWeight W, uint16_t *Y) {
    const int at = blockIdx.x * blockDim.x + threadIdx.x;                // word of a row
    if (at * 8 >= W.K) return;
    const int g = at >> 4, j = (at >> 2) & 3, t = at & 3;
    const uint8_t *codes = W.codes + static_cast<int64_t>(g) * kMxTileCodes + t * 16 + j * 4, *scales = W.scales + static_cast<int64_t>(g) * kMxTileScales + j;
    for (int m0 = blockIdx.y * kMxQuantRows; m0 < W.M; m0 += gridDim.y * kMxQuantRows) {
        uint32_t word[kMxQuantRows], scale[kMxQuantRows];
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) {                          // rows up to the end of a tile exist
            word[r] = __ldg(reinterpret_cast<const uint32_t *>(codes + mx_code_row(m0 + r, W.groups)));
            scale[r] = __ldg(scales + mx_scale_row(m0 + r, W.groups));
        }
#pragma unroll
        for (int r = 0; r < kMxQuantRows; r++) {
            float v[8];
            mx_word_to_f32(word[r], mx_scale(scale[r]), v);
            if (m0 + r < W.M)
                *reinterpret_cast<uint4 *>(Y + static_cast<int64_t>(m0 + r) * W.K + at * 8) =
                    make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
    }
}

// ---- the gated pair's gradient: dg = dh u act'(g), du = dh act(g) --------------------------------------------------------
// Bound by memory: 8 bytes of projections and 2 of dh in, 4 out.  A thread takes kVec neighbours of a row.  Everything up to the store is 32 bits
// wide; dg and du are rounded to BF16 because they are the operand of a BF16 product, of which no other type is exact on the expanded weight
// and as fast.  With the rounding of dx after it that makes the error of dx 0.0023 of its norm where one rounding makes 0.0017 (12288 x 4096, 2048 rows);
// two BF16 parts a value would take the product's time twice.
constexpr int kMxPairThreads = 256;

template <int kVec>
__global__ void __launch_bounds__(kMxPairThreads) mx_gated_grad_kernel(const float *pre, const uint16_t *dH, int act, uint16_t *dpre, int inter, int ldp, int rows) {
    const int c = (blockIdx.x * kMxPairThreads + threadIdx.x) * kVec;
    if (c >= inter) return;
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        const float *from = pre + static_cast<int64_t>(r) * 2 * inter + c;
        uint16_t *to = dpre + static_cast<int64_t>(r) * ldp + c;
        const uint16_t *dh = dH + static_cast<int64_t>(r) * inter + c;
        float g[kVec], u[kVec], d[kVec], dg[kVec], du[kVec];
        if constexpr (kVec == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4 *>(from)), b = __ldcs(reinterpret_cast<const float4 *>(from + inter));
            const uint2 h = __ldcs(reinterpret_cast<const uint2 *>(dh));
            g[0] = a.x, g[1] = a.y, g[2] = a.z, g[3] = a.w, u[0] = b.x, u[1] = b.y, u[2] = b.z, u[3] = b.w;
            d[0] = bf16lo_to_f32(h.x), d[1] = bf16hi_to_f32(h.x), d[2] = bf16lo_to_f32(h.y), d[3] = bf16hi_to_f32(h.y);
        } else {
            g[0] = from[0], u[0] = from[inter], d[0] = bf16lo_to_f32(dh[0]);
        }
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            float a, da;
            mx_act_grad(act, g[i], a, da);
            dg[i] = d[i] * u[i] * da;
            du[i] = d[i] * a;
        }
        if constexpr (kVec == 4) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16(dg[0], dg[1]), pack_bf16(dg[2], dg[3]));
            *reinterpret_cast<uint2 *>(to + inter) = make_uint2(pack_bf16(du[0], du[1]), pack_bf16(du[2], du[3]));
        } else {
            to[0] = f32_to_bf16_rn(dg[0]);
            to[inter] = f32_to_bf16_rn(du[0]);
        }
    }
}

// Does nothing, after a kernel that writes a weight: a kernel with launch overlap that follows may read the weight before it has waited for the kernel
// in front of it, which is then this one, and this one starts when the weight is complete.
__global__ void mx_settle_kernel() {}

// ---- host ----------------------------------------------------------------------------------------------------------------
static int mx_check(const void *codes, const void *scales, int M, int K) {
    BHI_REQUIRE(codes && scales, "null weight buffer");
    BHI_REQUIRE(M >= 1, "empty weight");
    BHI_REQUIRE(K >= 32 && K % 32 == 0, "columns must be a multiple of 32");
    BHI_REQUIRE(M <= BHI_MXFP4_MAX_DIM && K <= BHI_MXFP4_MAX_DIM, "weight dimension beyond the limit");
    BHI_REQUIRE(aligned(codes, 16) && aligned(scales, 16), "weight buffers must be 16-byte aligned");
    return BHI_OK;
}
static MxWeight mx_weight(const uint8_t *codes, const uint8_t *scales, int M, int K) { return {codes, scales, M, K, (K + kMxGroup - 1) / kMxGroup}; }

// Whether a product takes the kernel for few rows.  Its rate is the memory's where the weight is most of the traffic (16 rows: 12288 x 4096 14.0
// against 19.3 us, 4096 x 4096 8.9 against 10.3).  From nine rows on the tiles are faster where the weight is small (1024 x 1024, 9 rows 4.1
// against 5.9 us, 2048 x 2048 5.8 against 6.5; 4096 x 2048 7.4 against 6.7) and where every SM would read a large X for few outputs (2560 x
// 9728, 16 rows 14.0 against 20.3, 3584 x 18944, 9 rows 24.3 against 27.6; 2048 x 8192, 9 rows 11.8 against 10.1).  From 17 rows on ten steps an SM have to
// pay for X's conversion (24 rows: 24576 x 4096 33.6 against 34.3, 38000 x 12288 123 against 148, gated 18944 x 3584 36.8 against 36.2, at 20 rows 33.3
// against 36.1); with 32 rows nothing does (24576 x 4096 48 against 34).
static bool mx_few_rows(int rows, int M, int K) {
    if (rows <= 8) return true;
    if (rows > 16) return rows <= kMxRowsMost && M >= 160 * sm_count();
    if (static_cast<int64_t>(M) * K <= 1 << 22) return false;
    return static_cast<int64_t>(rows) * K <= 125000 || M > 22 * 256;
}

static int mx_launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BHI_OK : cuda_fail(e, what);
}
// Blocks and threads over the words of a row (whole warps, as few idle ones as possible) by rows, some eight blocks an SM.
static void mx_matrix_grid(int words, int M, dim3 &grid, dim3 &block) {
    const int across = (words + kMxQuantThreads - 1) / kMxQuantThreads;
    block = dim3(((words + across - 1) / across + 31) / 32 * 32);
    const int rows = (M + kMxQuantRows - 1) / kMxQuantRows, per_sm = 2048 / static_cast<int>(block.x), most = (sm_count() * per_sm * 2 + across - 1) / across;
    grid = dim3(across, rows < most ? rows : most);
}

}  // namespace bhi

using namespace bhi;

extern "C" {

int bhi_mxfp4_quantize(const void *W, int dtype, int M, int K, uint8_t *codes, uint8_t *scales, void *stream) {
    if (int rc = mx_check(codes, scales, M, K)) return rc;
    BHI_REQUIRE(W && aligned(W, 16), "the matrix must be 16-byte aligned");
    BHI_REQUIRE(dtype >= BHI_DTYPE_BF16 && dtype <= BHI_DTYPE_FP32, "unknown type");
    const int groups = (K + kMxGroup - 1) / kMxGroup;
    dim3 grid, block;
    mx_matrix_grid(groups * 16, (M + 15) / 16 * 16, grid, block);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
    case BHI_DTYPE_BF16: mx_quantize_kernel<<<grid, block, 0, st>>>(static_cast<const __nv_bfloat16 *>(W), M, K, groups, codes, scales); break;
    case BHI_DTYPE_FP16: mx_quantize_kernel<<<grid, block, 0, st>>>(static_cast<const __half *>(W), M, K, groups, codes, scales); break;
    default: mx_quantize_kernel<<<grid, block, 0, st>>>(static_cast<const float *>(W), M, K, groups, codes, scales); break;
    }
    mx_settle_kernel<<<1, 32, 0, st>>>();
    return mx_launched("quantisation launch");
}

int bhi_mxfp4_from_packed(const uint8_t *packed, const uint8_t *packed_scales, int M, int K, uint8_t *codes, uint8_t *scales, void *stream) {
    if (int rc = mx_check(codes, scales, M, K)) return rc;
    BHI_REQUIRE(packed && packed_scales && aligned(packed, 4), "packed codes must be 4-byte aligned");
    const int groups = (K + kMxGroup - 1) / kMxGroup;
    dim3 grid, block;
    mx_matrix_grid(groups * 16, (M + 15) / 16 * 16, grid, block);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    mx_layout_kernel<<<grid, block, 0, st>>>(packed, packed_scales, M, K, groups, codes, scales);
    mx_settle_kernel<<<1, 32, 0, st>>>();
    return mx_launched("layout launch");
}

int bhi_mxfp4_dense(const uint8_t *codes, const uint8_t *scales, int M, int K, uint16_t *Y, void *stream) {
    if (int rc = mx_check(codes, scales, M, K)) return rc;
    BHI_REQUIRE(Y && aligned(Y, 16), "the output must be 16-byte aligned");
    dim3 grid, block;
    mx_matrix_grid(K / 8, M, grid, block);
    mx_dense_kernel<<<grid, block, 0, static_cast<cudaStream_t>(stream)>>>(mx_weight(codes, scales, M, K), Y);
    return mx_launched("dense launch");
}

int bhi_mxfp4_linear(const uint8_t *codes, const uint8_t *scales, int M, int K, const uint16_t *X, const uint16_t *bias, uint16_t *Y, int rows,
                     void *stream) {
    if (int rc = mx_check(codes, scales, M, K)) return rc;
    BHI_REQUIRE(rows >= 1 && rows <= BHI_MXFP4_MAX_ROWS, "bad number of rows");
    BHI_REQUIRE(X && Y && aligned(X, 16) && aligned(Y, 2) && aligned(bias, 2), "X must be 16-byte aligned");
    if (mx_few_rows(rows, M, K)) {
        const int rc = mx_rows_launch(mx_weight(codes, scales, M, K), X, bias, Y, false, 0, nullptr, rows, static_cast<cudaStream_t>(stream));
        if (rc != kStagedDeclined) return rc;
    }
    return mx_tile_launch(mx_weight(codes, scales, M, K), X, bias, Y, false, 0, nullptr, rows, static_cast<cudaStream_t>(stream));
}

int bhi_mxfp4_linear_grad(const uint8_t *codes, const uint8_t *scales, int M, int K, const uint16_t *dY, int ldy, uint16_t *dX, int rows, void *stream) {
    if (int rc = mx_check(codes, scales, M, K)) return rc;
    BHI_REQUIRE(rows >= 1 && rows <= BHI_MXFP4_MAX_ROWS, "bad number of rows");
    BHI_REQUIRE(ldy >= M && ldy % 8 == 0, "rows of dY must be a multiple of 8 values apart");
    BHI_REQUIRE(dY && dX && aligned(dY, 16) && aligned(dX, 16), "dY and dX must be 16-byte aligned");
    return mx_grad_launch(mx_weight(codes, scales, M, K), dY, ldy, dX, rows, static_cast<cudaStream_t>(stream));
}

int bhi_mxfp4_gated(const uint8_t *codes, const uint8_t *scales, int inter, int K, const uint16_t *X, const uint16_t *bias, int activation, uint16_t *H,
                    float *pre, int rows, void *stream) {
    BHI_REQUIRE(inter >= 1 && inter <= BHI_MXFP4_MAX_DIM / 2, "bad number of gated outputs");
    if (int rc = mx_check(codes, scales, 2 * inter, K)) return rc;
    BHI_REQUIRE(rows >= 1 && rows <= BHI_MXFP4_MAX_ROWS, "bad number of rows");
    BHI_REQUIRE(activation >= BHI_ACT_SILU && activation <= BHI_ACT_GELU_TANH, "unknown activation");
    BHI_REQUIRE(X && H && aligned(X, 16) && aligned(H, 2) && aligned(bias, 2) && aligned(pre, 16), "X must be 16-byte aligned");
    const MxWeight W = mx_weight(codes, scales, 2 * inter, K);
    if (mx_few_rows(rows, W.M, K)) {
        const int rc = mx_rows_launch(W, X, bias, H, true, activation, pre, rows, static_cast<cudaStream_t>(stream));
        if (rc != kStagedDeclined) return rc;
    }
    return mx_tile_launch(W, X, bias, H, true, activation, pre, rows, static_cast<cudaStream_t>(stream));
}

int bhi_mxfp4_gated_grad(const float *pre, const uint16_t *dH, int inter, int activation, uint16_t *dpre, int ldp, int rows, void *stream) {
    BHI_REQUIRE(inter >= 1 && inter <= BHI_MXFP4_MAX_DIM / 2 && rows >= 1 && rows <= BHI_MXFP4_MAX_ROWS, "bad size of a gated gradient");
    BHI_REQUIRE(pre && dH && dpre && aligned(pre, 16) && aligned(dH, 2) && aligned(dpre, 16) && ldp >= 2 * inter && ldp % 4 == 0, "bad gradient buffers");
    BHI_REQUIRE(activation >= BHI_ACT_SILU && activation <= BHI_ACT_GELU_TANH, "unknown activation");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = inter % 4 == 0 && aligned(dH, 8);
    const int across = (inter + kMxPairThreads * (wide ? 4 : 1) - 1) / (kMxPairThreads * (wide ? 4 : 1)), most = (sm_count() * 16 + across - 1) / across;
    const dim3 grid(across, rows < most ? rows : most);
    if (wide) mx_gated_grad_kernel<4><<<grid, kMxPairThreads, 0, st>>>(pre, dH, activation, dpre, inter, ldp, rows);
    else mx_gated_grad_kernel<1><<<grid, kMxPairThreads, 0, st>>>(pre, dH, activation, dpre, inter, ldp, rows);
    return mx_launched("gated gradient launch");
}

}  // extern "C"
