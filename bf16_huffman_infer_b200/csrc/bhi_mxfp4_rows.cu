// The products of 4-bit microscaled weights with few rows of X: which form, and its launch.
#include <algorithm>

#include "bhi_mxfp4_rows.cuh"

namespace bhi {

bool overlap_launches();

namespace {

constexpr uint32_t kSmemRows = kSmemMax - 1024;      // what the barriers leave
constexpr uint32_t kSmemHalf = 112 * 1024;           // of two CTAs an SM
constexpr int kChunksMax = 8;

template <class Form>
int launch(MxRowsArgs a, cudaStream_t st) {
    constexpr int per = Form::kGated ? 8 : 16 * Form::MT;
    a.steps = (a.outs + per - 1) / per;
    const int groups = a.W.groups, grid = std::min(a.steps, sm_count() * Form::kPerSm), most_steps = (a.steps + grid - 1) / grid;
    // as few chunks of K as shared memory takes
    for (int chunks = 1; chunks <= (Form::kPerSm == 2 ? 1 : kChunksMax) && chunks <= groups; chunks++) {
        a.chunk_groups = (groups + chunks - 1) / chunks;
        a.scale_off = static_cast<uint32_t>(a.rows) * Form::row_bytes(a.chunk_groups);
        a.part_off = a.scale_off + (Form::kHalf ? static_cast<uint32_t>(a.chunk_groups) * 8 * Form::NT * 4 : 0u);
        a.sum_off = a.part_off + Form::kWarps * Form::kPlaces * Form::kPart * 16u;
        const uint64_t bytes = a.sum_off + (chunks > 1 ? static_cast<uint64_t>(most_steps) * Form::kPart * 16u : 0u);
        if (bytes > (Form::kPerSm == 2 ? kSmemHalf : kSmemRows)) continue;
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
    if (gated && rows > 8) return launch<MxRowsForm<1, 2, 16, 1, 4, true>>(a, st);
    if (gated) {
        // as below; from five rows on one CTA an SM, which brings and converts X once (18944 x 3584, 8 rows 20.2 against 22.5 us)
        const int rc = rows <= 4 ? launch<MxRowsForm<1, 1, 8, 2, 3, true>>(a, st) : kStagedDeclined;
        return rc != kStagedDeclined ? rc : launch<MxRowsForm<1, 1, 16, 1, 3, true>>(a, st);
    }
    if (rows > 8) return launch<MxRowsForm<1, 2, 16, 1, 4, false>>(a, st);
    // Two CTAs an SM, so that the next kernel's are there as soon as one of them ends, where X leaves them room; two tiles a step share X's
    // fragments (151936 x 4096, 8 rows 65.7 against 72 us) where every CTA has four steps of them (37984 x 4096 either way 24).
    const int rc = W.M >= 128 * 2 * sm_count() ? launch<MxRowsForm<2, 1, 8, 2, 2, false>>(a, st) : launch<MxRowsForm<1, 1, 8, 2, 4, false>>(a, st);
    return rc != kStagedDeclined ? rc : launch<MxRowsForm<1, 1, 16, 1, 4, false>>(a, st);
}

cudaError_t take_mxfp4_rows_status(int *out) { return take_status(out); }

}  // namespace bhi
