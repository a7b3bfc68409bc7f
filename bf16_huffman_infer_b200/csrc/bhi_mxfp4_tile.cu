// The products of 4-bit microscaled weights in tiles: plans and launches.
#include <mutex>

#include "bhi_mxfp4_tile.cuh"

namespace bhi {

bool overlap_launches();

namespace {

constexpr uint32_t kSmemTile = kSmemMax - 1024;      // what the barriers leave
constexpr int kSplitsMost = 4;                       // clusters of eight CTAs

// The tensor-map encoder lives in the driver library, which this library does not link: it is looked up through the runtime once.
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

enum Kind { kPlain, kGatedPair, kGradient };

// How many clusters of `splits` pairs of CTAs are active at a time (of 74 pairs of SMs 33 twos, 22 threes, 15 fours: a cluster lies in one GPC).
int clusters_that_fit(int splits) {
    static std::mutex mu;
    static int cached[64][kSplitsMost + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    std::lock_guard<std::mutex> lock(mu);
    int &n = cached[dev][splits];
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sm_count() / (2 * splits) * (2 * splits));
        cfg.blockDim = dim3(kMtThreads);
        cfg.dynamicSmemBytes = kSmemTile;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2 * splits;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (staged_prepare(mx_grad_kernel, kSmemTile) != BHI_OK || cudaOccupancyMaxActiveClusters(&n, mx_grad_kernel, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = -1;                              // none
        }
    }
    return n;
}

// Rows of a tile (a multiple of 32), and into how many parts c is cut (up to four pairs of SMs share a tile): the fewest rounds of tiles over
// the pairs of SMs times what a tile costs, by its rows: measured (4096 columns, ns for 128 of them) 425 + 0.85 rows forward, twice (395 + 0.55
// rows) for a gradient.  An accumulator on its own (above 128 rows, forward) keeps the products waiting while it is read; the
// sums of parts take their way through shared memory (1000 + 16.5 rows), and parts run in one round only, of the clusters that fit.  (A last round's few tiles as a
// launch of their own, in parts: 37984 x 4096, 64 rows, 149 tiles 48 against 51 us, but gated 12288 x 4096, 2048 rows, 768 tiles no faster.)
struct TilePlan {
    int nt = 32, splits = 1;
};
TilePlan tile_plan(int rows, int pairs_p, int groups, bool gradient) {
    TilePlan best;
    double best_cost = 1e30;
    const int pairs = sm_count() / 2;
    for (int nt = 32; nt <= kMtRows; nt += 32) {
        const int64_t tiles = static_cast<int64_t>((rows + nt - 1) / nt) * pairs_p;
        const double group = gradient ? 2 * (395 + 0.55 * nt) : 425 + 0.85 * nt;
        for (int s = 1; s <= kSplitsMost; s++) {
            if (s > 1 && (tiles > clusters_that_fit(s) || groups < 2 * s)) break;
            const double rounds = static_cast<double>((tiles + pairs - 1) / pairs);
            const double tile = (groups + s - 1) / s * group + (s == 1 ? nt > kMtTwoRows && !gradient ? 6.0 * nt : 0.0 : 1000 + 16.5 * nt);
            if (rounds * tile + 1e-3 * nt < best_cost - 1e-9) {
                best_cost = rounds * tile + 1e-3 * nt;
                best.nt = nt;
                best.splits = s;
            }
        }
        if (nt >= rows) break;
    }
    return best;
}

template <Kind kKind>
int launch(MxTileArgs a, const uint16_t *B, int64_t b_cols, int64_t ldb, cudaStream_t st) {
    EncodeTiledFn encode = encode_tiled();
    if (!encode) return fail(BHI_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const int per = kKind == kGatedPair ? 64 : 128;
    a.pairs_p = (a.outs + 2 * per - 1) / (2 * per);
    const TilePlan plan = tile_plan(a.rows, a.pairs_p, static_cast<int>((b_cols + 127) / 128), kKind == kGradient);
    a.nt = plan.nt;
    a.splits = plan.splits;
    a.tiles_n = (a.rows + a.nt - 1) / a.nt;
    a.buffers = kKind == kGradient || a.nt <= kMtTwoRows ? 2 : 1;
    a.boxes_c = static_cast<int>((b_cols + kMtBox - 1) / kMtBox);
    const int whole = kKind == kGradient ? 1 : 2, units = (a.boxes_c + whole - 1) / whole;      // a group forward
    a.split_boxes = (units + a.splits - 1) / a.splits * whole;
    if (a.split_boxes * (a.splits - 1) >= a.boxes_c) a.splits = 1, a.split_boxes = a.boxes_c;
    BHI_REQUIRE(static_cast<int64_t>(a.pairs_p) * a.tiles_n <= INT32_MAX / 2, "too many tiles");
    const uint32_t stage = kKind == kGradient ? kMtABytes + static_cast<uint32_t>(a.nt) * 64u : static_cast<uint32_t>(a.nt) * 128u, extra = kKind == kGradient ? 0u : static_cast<uint32_t>(a.nt) * 512u;      // sums
    a.stages = static_cast<int>((kSmemTile - extra) / stage);
    if (a.stages > kMtStagesMax) a.stages = kMtStagesMax;
    if (kKind == kGradient) a.stages &= ~1;          // a slot is always the same team's
    const int vec = kKind == kGatedPair ? 2 : 4;
    a.wide = a.outs % vec == 0 && aligned(a.out, 2 * vec);
    alignas(64) CUtensorMap map;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(b_cols), static_cast<cuuint64_t>(a.rows)}, strides[1] = {static_cast<cuuint64_t>(ldb) * 2};
    const cuuint32_t box[2] = {kMtBox, static_cast<cuuint32_t>(a.nt / 2)}, estr[2] = {1, 1};
    const auto encoded = [&]() {
        return encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t *>(B), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult cr = encoded();
    if (cr == CUDA_ERROR_INVALID_CONTEXT) {          // a thread that has not called the runtime yet (an autograd thread): bind the device's context
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) cr = encoded();
    }
    if (cr != CUDA_SUCCESS) return fail(BHI_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(cr)));
    auto kernel = kKind == kGradient ? mx_grad_kernel : mx_tile_kernel<kKind == kGatedPair>;
    if (int rc = staged_prepare(kernel, kSmemTile)) return rc;
    const int tiles = a.pairs_p * a.tiles_n, pairs = sm_count() / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * a.splits * (tiles < pairs ? tiles : pairs));
    cfg.blockDim = dim3(kMtThreads);
    cfg.dynamicSmemBytes = a.stages * stage + extra;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * a.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_launches() ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, map);
    return e == cudaSuccess ? BHI_OK : cuda_fail(e, "4-bit tiled product launch");
}

}  // namespace

int mx_tile_launch(const MxWeight &W, const uint16_t *X, const uint16_t *bias, uint16_t *Y, bool gated, int activation, float *pre, int rows, cudaStream_t st) {
    MxTileArgs a{};
    a.W = W, a.bias = bias, a.out = Y, a.pre = pre, a.rows = rows, a.outs = gated ? W.M / 2 : W.M, a.activation = activation;
    return gated ? launch<kGatedPair>(a, X, W.K, W.K, st) : launch<kPlain>(a, X, W.K, W.K, st);
}

int mx_grad_launch(const MxWeight &W, const uint16_t *dY, int ldy, uint16_t *dX, int rows, cudaStream_t st) {
    MxTileArgs a{};
    a.W = W, a.out = dX, a.rows = rows, a.outs = W.K;
    return launch<kGradient>(a, dY, W.M, ldy, st);
}

cudaError_t take_mxfp4_tile_status(int *out) { return take_status(out); }

}  // namespace bhi
