// The products of 4-bit microscaled weights with few rows of X: which form, and its launch.
#include <algorithm>

#include "bhi_mxfp4_rows.cuh"

namespace bhi {

bool overlap_launches();

namespace {

constexpr uint32_t kSmemRows = kSmemMax - 1024;      // what the barriers leave
constexpr int kChunksMax = 8;

template <class Form>
int launch(MxRowsArgs a, cudaStream_t st) {
    constexpr int per = Form::kGated ? 8 : 16 * Form::MT;
    a.steps = (a.outs + per - 1) / per;
    const int groups = a.W.groups, grid = std::min(a.steps, sm_count() * Form::kPerSm), most_steps = (a.steps + grid - 1) / grid;
    // as few chunks of K as shared memory takes
    for (int chunks = 1; chunks <= kChunksMax && chunks <= groups; chunks++) {
        a.chunk_groups = (groups + chunks - 1) / chunks;
        a.scale_off = static_cast<uint32_t>(a.rows) * Form::row_bytes(a.chunk_groups);
        a.part_off = a.scale_off + (Form::kHalf ? static_cast<uint32_t>(a.chunk_groups) * 8 * Form::NT * 4 : 0u);
        a.sum_off = a.part_off + Form::kWarps * Form::kPlaces * Form::kPart * 16u;
        const uint64_t bytes = a.sum_off + (chunks > 1 ? static_cast<uint64_t>(most_steps) * Form::kPart * 16u : 0u);
        if (bytes > kSmemRows) continue;
        auto kernel = mx_rows_kernel<Form>;
        if (int rc = staged_prepare(kernel, kSmemRows)) return rc;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(Form::kThreads);
        cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = overlap_launches() ? 1 : 0;
        cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
        return e == cudaSuccess ? BHI_OK : cuda_fail(e, "4-bit product launch");
    }
    return kStagedDeclined;
}

}  // namespace

int mx_rows_launch(const MxWeight &W, const uint16_t *X, const uint16_t *bias, uint16_t *Y, bool gated, int activation, float *pre, int rows, cudaStream_t st) {
    // the kernel counts a weight's codes in pieces of 16 bytes, 32 bits wide
    if (rows > kMxRowsMost || static_cast<int64_t>((W.M + 15) / 16) * W.groups * (kMxTileCodes / 16) > UINT32_MAX) return kStagedDeclined;
    MxRowsArgs a{};
    a.W = W, a.X = X, a.bias = bias, a.Y = Y, a.pre = pre, a.rows = rows, a.outs = gated ? W.M / 2 : W.M, a.activation = activation;
    if (rows > 16) return gated ? launch<MxRowsForm<1, 3, 16, 1, 2, true>>(a, st) : launch<MxRowsForm<1, 3, 16, 1, 2, false>>(a, st);
    if (rows > 8) {
        // FP16 where an SM has ten steps or more (16 rows: 151936 x 4096 85 against 108 us, 64 steps; 32000 x 4096 25.3 against 26.9, 13; gated 12288 x
        // 4096 23.1 both, ten; 12288 x 4096 16.2 against 14.0, five; gated 4096 x 2048 9.3 against 7.6, three)
        const bool half = (a.outs + (gated ? 7 : 15)) / (gated ? 8 : 16) >= 10 * sm_count();
        if (gated) return half ? launch<MxRowsForm<1, 2, 16, 1, 3, true>>(a, st) : launch<MxRowsForm<1, 2, 16, 1, 4, true, false>>(a, st);
        return half ? launch<MxRowsForm<1, 2, 16, 1, 3, false>>(a, st) : launch<MxRowsForm<1, 2, 16, 1, 4, false, false>>(a, st);
    }
    if (gated) return launch<MxRowsForm<1, 1, 16, 1, 3, true>>(a, st);
    // Two tiles a step share X's fragments (151936 x 4096, 8 rows 62 against 65 us; fewer steps: 37984 x 4096, 8 rows 21.7 against 20.9) where every SM
    // has eight steps of them.  Where X is small, two CTAs an SM: the next kernel's are there as soon as one of them ends (1 row: 4096 x 4096 6.1 against
    // 6.7 us, 37984 x 4096 19.5 against 20.0); else one, which brings and converts X once (4096 x 12288, 1 row 10.8 against 11.4; 12288 x 4096, 8 rows
    // 11.4 against 14.2).
    const bool many = W.M >= 256 * sm_count();
    if (static_cast<int64_t>(rows) * W.K <= 8192) return many ? launch<MxRowsForm<2, 1, 8, 2, 2, false>>(a, st) : launch<MxRowsForm<1, 1, 8, 2, 4, false>>(a, st);
    return many ? launch<MxRowsForm<2, 1, 16, 1, 2, false>>(a, st) : launch<MxRowsForm<1, 1, 16, 1, 4, false>>(a, st);
}

cudaError_t take_mxfp4_rows_status(int *out) { return take_status(out); }

}  // namespace bhi
