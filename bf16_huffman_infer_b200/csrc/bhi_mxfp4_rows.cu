// The products of 4-bit microscaled weights with few rows of X: which form, and its launch.
#include <algorithm>
#include <cstdlib>

#include "bhi_mxfp4_rows.cuh"

namespace bhi {

bool overlap_launches();

namespace {

constexpr uint32_t kSmemRows = kSmemMax - 1024;      // what the barriers leave
constexpr uint32_t kSmemHalf = 112 * 1024;           // of two CTAs an SM
constexpr int kChunksMax = 8;

template <class Form>
int launch(MxRowsArgs a, cudaStream_t st) {
    constexpr int per = Form::kGated ? 16 : 16 * Form::MT;
    a.steps = (a.outs + per - 1) / per;
    const int groups = a.W.groups, grid = std::min(a.steps, sm_count() * Form::kPerSm), most_steps = (a.steps + grid - 1) / grid;
    // as few chunks of K as shared memory takes
    for (int chunks = 1; chunks <= (Form::kPerSm == 2 ? 1 : kChunksMax) && chunks <= groups; chunks++) {
        a.chunk_groups = (groups + chunks - 1) / chunks;
        const int last = groups - (groups - 1) / a.chunk_groups * a.chunk_groups;      // groups of the last chunk
        a.consumers = std::min(Form::kWarps, last);
        a.scale_off = static_cast<uint32_t>(a.rows) * Form::row_bytes(a.chunk_groups);
        a.part_off = a.scale_off + static_cast<uint32_t>(a.chunk_groups) * 8 * Form::NT * 4;
        for (a.parts = kMxPartsMax; a.parts >= 2; a.parts--) {
            a.sum_off = a.part_off + a.parts * a.consumers * Form::kPart * 16u;
            const uint64_t bytes = a.sum_off + (chunks > 1 ? static_cast<uint64_t>(most_steps) * Form::kSum * 16u : 0u);
            if (bytes > (Form::kPerSm == 2 ? kSmemHalf : kSmemRows)) continue;
            auto kernel = mx_rows_kernel<Form>;
            if (int rc = staged_prepare(kernel, kSmemRows)) return rc;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(grid);
            cfg.blockDim = dim3(32 * (a.consumers + Form::kFinishers));
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
    }
    return kStagedDeclined;
}

}  // namespace

int mx_rows_launch(const MxWeight &W, const uint16_t *X, const uint16_t *bias, uint16_t *Y, bool gated, int activation, float *pre, int rows, cudaStream_t st) {
    MxRowsArgs a{};
    a.W = W, a.X = X, a.bias = bias, a.Y = Y, a.pre = pre, a.rows = rows, a.outs = gated ? W.M / 2 : W.M, a.activation = activation;
    static const int f = getenv("MXF") ? atoi(getenv("MXF")) : 0;
    if (gated && a.outs % 16 == 0) {
        if (f == 1 && rows <= 8) return launch<MxRowsForm<2, 1, 18, 2, 1, 1, true>>(a, st);
        if (f == 1 && rows <= 16) return launch<MxRowsForm<2, 2, 18, 2, 1, 1, true>>(a, st);
        if (f == 2 && rows <= 16) return launch<MxRowsForm<2, 2, 22, 2, 1, 1, true>>(a, st);
        if (rows <= 8) return launch<MxRowsForm<2, 1, 14, 2, 1, 2, true>>(a, st);
        if (rows <= 16) return launch<MxRowsForm<2, 2, 14, 2, 1, 2, true>>(a, st);
        if (rows <= 32) return launch<MxRowsForm<2, 4, 14, 2, 1, 1, true>>(a, st);
    } else if (gated) {                              // ups lie across two tiles each
        if (rows <= 8) return launch<MxRowsForm<3, 1, 14, 2, 1, 1, true>>(a, st);
        if (rows <= 16) return launch<MxRowsForm<3, 2, 14, 2, 1, 1, true>>(a, st);
        if (rows <= 32) return launch<MxRowsForm<3, 4, 10, 2, 1, 1, true>>(a, st);
    } else {
        int rc = kStagedDeclined;
        if (rows <= 8) rc = W.M >= 128 * 2 * sm_count() ? launch<MxRowsForm<2, 1, 7, 1, 2, 2, false>>(a, st) : launch<MxRowsForm<1, 1, 7, 1, 2, 4, false>>(a, st);
        if (rc != kStagedDeclined) return rc;
        if (f == 1 && rows <= 16) return launch<MxRowsForm<2, 2, 18, 2, 1, 1, false>>(a, st);
        if (f == 2 && rows <= 16) return launch<MxRowsForm<1, 2, 18, 2, 1, 3, false>>(a, st);
        if (f == 3 && rows <= 16) return launch<MxRowsForm<1, 2, 22, 2, 1, 2, false>>(a, st);
        if (f == 1 && rows <= 32) return launch<MxRowsForm<2, 4, 14, 2, 1, 1, false>>(a, st);
        if (f == 2 && rows <= 32) return launch<MxRowsForm<1, 4, 18, 2, 1, 2, false>>(a, st);
        if (rows <= 8) return launch<MxRowsForm<2, 1, 14, 2, 1, 2, false>>(a, st);
        if (rows <= 16) return launch<MxRowsForm<2, 2, 14, 2, 1, 2, false>>(a, st);
        if (rows <= 32) return launch<MxRowsForm<1, 4, 14, 2, 1, 2, false>>(a, st);
    }
    return kStagedDeclined;
}

cudaError_t take_mxfp4_rows_status(int *out) { return take_status(out); }

}  // namespace bhi
