// 4-bit microscaled weights (OCP MXFP4): the layout in memory and what every kernel on them shares.
//
// Blocks of 32 values along a row share a scale byte s (E8M0, 2^(s - 127); 255 is NaN); a value is a 4-bit code (E2M1: sign,
// two exponent bits, one mantissa bit; 0, 0.5, 1, 1.5, 2, 3, 4, 6).
//
// The rows are cut into tiles of 16 and the columns into groups of 128; both are padded with zeros.  One (tile, group) pair is
// 1 KB of codes and 64 bytes of scales, so whatever walks along K reads whole lines.  A lane of an m16n8k16 product finds the four
// words it needs of a row in one 16-byte load, and the eight lanes that a load is served by at a time, two rows of four, read one line.  (With a
// quarter's rows side by side they read four, and the first level's data path bounded the kernel: 151936 x 4096, 1 row 62.0 against 59.8 us;
// readers that take a row a lane would have it so: 37984 x 4096, 64 rows 49.6 against 51.4.)
//
//   codes  [ceil(M / 16)][ceil(K / 128)][16 rows][4 quarters t][4 blocks j][4 bytes]   word (t, j): elements 8 t .. 8 t + 7 of block j
//   scales [ceil(M / 16)][ceil(K / 128)][16 rows][4 blocks j]
//
// Inside a word, nibble i is element 2 i and nibble 4 + i element 2 i + 1 (i = 0..3): a mask leaves the pair (2 i, 2 i + 1) in
// the two halves of a register.  Blocks whose scale is NaN hold zero codes, so that a product with an infinite scale yields NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "bhi_staged.cuh"

namespace bhi {

constexpr int kMxRows = 16;                     // rows of a tile
constexpr int kMxGroup = 128;                   // columns of a group
constexpr int kMxTileCodes = 1024;              // bytes of a (tile, group) pair
constexpr int kMxTileScales = 64;
constexpr int kMxRowCodes = 64;                 // bytes of a row in it

struct MxWeight {
    const uint8_t *codes, *scales;
    int M, K, groups;                           // groups = ceil(K / 128)
};

// byte offsets of row m, group 0
__host__ __device__ __forceinline__ int64_t mx_code_row(int m, int groups) {
    return static_cast<int64_t>(m >> 4) * groups * kMxTileCodes + (m & 15) * kMxRowCodes;
}
__host__ __device__ __forceinline__ int64_t mx_scale_row(int m, int groups) {
    return static_cast<int64_t>(m >> 4) * groups * kMxTileScales + (m & 15) * 4;
}

// A wait of at most about a second, counted from the end of the kernel before (which has its own limits, more than one of them: for a peer's
// signals, say) where this one runs ahead of it.  When one runs out, the kernel's status word is set and no other wait of the CTA goes on: the
// CTA runs to its end with whatever it has.
__device__ __forceinline__ void mx_wait(uint32_t bar, uint32_t parity, int *dead, int status) {
    uint64_t t0 = 0;
    for (uint32_t i = 1; !mbar_try_wait(bar, parity); i++) {
        if ((i & 1023u) != 0u) continue;
        if (*static_cast<volatile int *>(dead)) return;
        if (t0 == 0) pdl_wait(), t0 = global_ns();
        const uint64_t now = global_ns();
        if (now - t0 > 1000000000ull) {
            atomicExch(dead, 1);
            atomicExch(&g_staged_status, status);
            return;
        }
    }
}

// Byte b of a code word as two FP16 values: nibble 2 b in the low half, 2 b + 1 in the high half.
__device__ __forceinline__ void mx_word_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

// Four scale bytes as BF16 pairs; 255 becomes NaN.
__device__ __forceinline__ void mx_scales_bf16(uint32_t s, uint32_t (&p)[2]) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.bf16x2.ue8m0x2 %0, l;\n\tcvt.rn.bf16x2.ue8m0x2 %1, h;\n\t}" : "=r"(p[0]), "=r"(p[1]) : "r"(s));
}

__device__ __forceinline__ float f16lo_to_f32(uint32_t pair) {
    float f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;\n\t}" : "=f"(f) : "r"(pair));
    return f;
}
__device__ __forceinline__ float f16hi_to_f32(uint32_t pair) {
    float f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, h;\n\t}" : "=f"(f) : "r"(pair));
    return f;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// A code's bits s eem are moved to a BF16's sign, lowest exponent and highest mantissa bits: that is its value times 2^-126, the
// subnormal code 0.5 included, and one product by 2^(126 + s - 127) makes both the value and its scale.  Scales above 2 (2^(126 + s - 127) would
// overflow) take two products.
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Eight codes as eight BF16 values in element order, times f (kLarge: times 2^126, then f).
template <bool kLarge>
__device__ __forceinline__ uint4 mx_word_to_bf16(uint32_t w, uint32_t f) {
    constexpr uint32_t kMag = 0x01C001C0u, kSign = 0x80008000u;
    uint32_t h[4];
    h[0] = ((w << 6) & kMag) | ((w << 12) & kSign);
    h[1] = ((w << 2) & kMag) | ((w << 8) & kSign);
    h[2] = ((w >> 2) & kMag) | ((w << 4) & kSign);
    h[3] = ((w >> 6) & kMag) | (w & kSign);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = mul_bf16x2(kLarge ? mul_bf16x2(h[i], 0x7E807E80u) : h[i], f);
    return make_uint4(h[0], h[1], h[2], h[3]);
}
// The factors of a row's four blocks: 2^(s - 1), or of large scales 2^(s - 127) (255: infinity, and its codes are zero).
template <bool kLarge>
__device__ __forceinline__ void mx_factors(uint32_t scales, uint32_t (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t s = (scales >> (8 * j)) & 255u;
        f[j] = kLarge ? (s == 0u ? 0x00400040u : s * 0x00800080u) : s * 0x00800080u + 0x3F003F00u;
    }
}
__device__ __forceinline__ uint32_t word_of(const uint4 &q, int j) { return j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w; }

// 2^(s - 127); 255 gives infinity here (its codes are zero, so that their product is NaN)
__device__ __forceinline__ float mx_scale(uint32_t s) { return __uint_as_float(s == 0u ? 0x00400000u : s << 23); }

// The eight values of a word in element order, exact in 32 bits.
__device__ __forceinline__ void mx_word_to_f32(uint32_t w, float scale, float (&v)[8]) {
    uint32_t h[4];
    mx_word_to_f16(w, h);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        // halves of h[i] are nibbles 2 i and 2 i + 1, and nibble n is element 2 n (n < 4) or 2 (n - 4) + 1
        const int n = 2 * i;
        v[n < 4 ? 2 * n : 2 * (n - 4) + 1] = f16lo_to_f32(h[i]) * scale;
        v[n + 1 < 4 ? 2 * (n + 1) : 2 * (n - 3) + 1] = f16hi_to_f32(h[i]) * scale;
    }
}

// ---- activations of the gated pair ---------------------------------------------------------------------------------
// act(g) = g s(g) and act'(g), in 32 bits.  s is a logistic function (silu: of g; gelu's tanh form: of 2 z, since
// (1 + tanh z) / 2 = 1 / (1 + exp(-2 z)), which does not cancel for negative z) or half of erfc(-g / sqrt 2).  The fast exponential
// and division are off by a few units of 2^-23 here: far below the one rounding to BF16 that follows.
__device__ __forceinline__ float mx_logistic(float v) {
    const float e = __expf(-fabsf(v));                                       // at most 1, and the tail of negative v keeps its digits
    return __fdividef(v < 0.f ? e : 1.f, 1.f + e);
}

__device__ __forceinline__ void mx_act_grad(int act, float g, float &a, float &da) {
    if (act == BHI_ACT_SILU) {
        const float s = mx_logistic(g);
        a = g * s;
        da = s + a * (1.f - s);
    } else if (act == BHI_ACT_GELU) {
        const float c = 0.5f * erfcf(g * -0.70710678118654752f);
        a = g * c;
        da = c + g * 0.39894228040143268f * __expf(-0.5f * g * g);
    } else {
        const float g2 = g * g;
        const float s = mx_logistic(1.59576912160573071f * (g + 0.044715f * g2 * g));
        a = g * s;
        da = s + a * (1.f - s) * 1.59576912160573071f * (1.f + 0.134145f * fminf(g2, 1e4f));      // beyond, a (1 - s) is zero, or would be times infinity
    }
}
__device__ __forceinline__ float mx_act(int act, float g) {
    if (act == BHI_ACT_SILU) return g * mx_logistic(g);
    if (act == BHI_ACT_GELU) return g * (0.5f * erfcf(g * -0.70710678118654752f));
    return g * mx_logistic(1.59576912160573071f * (g + 0.044715f * g * g * g));
}

// Rows of X that the kernel which reads the weight straight into registers takes at most.
constexpr int kMxRowsMost = 24;

// The products' launchers, whose source files are compiled side by side.  Each returns kStagedDeclined for what it does not serve.
// `gated`: W.M = 2 * outputs; pre may be null.
int mx_rows_launch(const MxWeight &W, const uint16_t *X, const uint16_t *bias, uint16_t *Y, bool gated, int activation, float *pre, int rows, cudaStream_t st);
int mx_tile_launch(const MxWeight &W, const uint16_t *X, const uint16_t *bias, uint16_t *Y, bool gated, int activation, float *pre, int rows, cudaStream_t st);
int mx_grad_launch(const MxWeight &W, const uint16_t *dY, int ldy, uint16_t *dX, int rows, cudaStream_t st);

}  // namespace bhi
