// The products of 4-bit microscaled weights with few rows of X: which form, and its launch.
#include "bhi_mxfp4_rows.cuh"

namespace bhi {

bool overlap_launches();

namespace {

// The CTAs that share a step's columns (a cluster of 1, 2, 4 or 8): the fewest rounds of units, a cluster's joins counted as kJoin
// units.
struct RowsPlan {
    int cluster = 0, part_groups = 0, clusters = 0;
    uint32_t smem = 0;
};
constexpr double kJoin = 1.5;

template <int NT>
RowsPlan rows_plan(int steps, int groups, int rows) {
    RowsPlan best;
    double best_cost = 1e30;
    for (int c = 1; c <= kMxClusterMax && c <= groups; c *= 2) {
        const int part = (groups + c - 1) / c;
        const uint32_t smem = MxRowsPlan<NT>::total(rows, part, c);
        if (smem > static_cast<uint32_t>(kSmemMax)) continue;
        const int per_sm = smem <= 113u * 1024u ? 2 : 1;
        const int clusters = sm_count() * per_sm / c;
        const int rounds = (steps + clusters - 1) / clusters, units = (part + kMxRowWarps - 1) / kMxRowWarps;
        const double cost = static_cast<double>(rounds) * units * per_sm + (c > 1 ? kJoin * ((rounds + kMxBatch - 1) / kMxBatch) : 0.0);
        if (cost < best_cost - 1e-9) {
            best_cost = cost;
            best = {c, part, steps < clusters ? steps : clusters, smem};
        }
    }
    return best;
}

template <int NT, int kDepth, bool kGated>
int launch(MxRowsArgs a, cudaStream_t st) {
    const RowsPlan p = rows_plan<NT>(a.steps, a.W.groups, a.rows);
    if (p.cluster == 0) return kStagedDeclined;
    auto kernel = mx_rows_kernel<NT, kDepth, kGated>;
    if (int rc = staged_prepare(kernel)) return rc;
    a.part_groups = p.part_groups;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.clusters * p.cluster);
    cfg.blockDim = dim3(kMxRowThreads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (overlap_launches()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (p.cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = p.cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e == cudaSuccess ? BHI_OK : cuda_fail(e, "4-bit product launch");
}

}  // namespace

int mx_rows_launch(const MxWeight &W, const uint16_t *X, const uint16_t *bias, uint16_t *Y, bool gated, int activation, float *pre, int rows, cudaStream_t st) {
    const int outs = gated ? W.M / 2 : W.M, per = gated ? 8 : 16;
    const MxRowsArgs a{W, X, bias, Y, pre, rows, outs, (outs + per - 1) / per, 0, activation};
    if (rows <= 8) return gated ? launch<1, 4, true>(a, st) : launch<1, 4, false>(a, st);
    if (rows <= 16) return gated ? launch<2, 4, true>(a, st) : launch<2, 4, false>(a, st);
    if (rows <= 32) return gated ? launch<4, 2, true>(a, st) : launch<4, 2, false>(a, st);
    return kStagedDeclined;
}

}  // namespace bhi
