// Host side of the layer operators around the grouped GEMM: argument checks, workspaces and launches
// of the router, dispatch / combine and the 4-bit products (C ABI in include/gg_b200.h).
//
// As with the grouped GEMM, a prepare call validates the problem and allocates what the handle needs,
// and gg_run enqueues the prepared operator's kernels without waiting.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <new>

#include "gg_b200.h"
#include "gg_handle.h"
#include "gg_permute.cuh"
#include "gg_route.cuh"
#include "gg_w4.cuh"

namespace gg {

int run_moe(gg_handle *h, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    // as in gg_run: every kernel waits for the one before it before it touches global memory
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = stream;
    void *args[2] = {&h->moe.map, h->moe.params};
    for (int i = 0; i < h->moe.launches; ++i) {
        const MoeLaunch &l = h->moe.launch[i];
        if (!l.grid)
            continue;  // nothing to do
        cfg.gridDim = dim3(l.grid, l.grid_y, 1);
        cfg.blockDim = dim3(l.block, 1, 1);
        cfg.dynamicSmemBytes = l.smem;
        attr[0].val.clusterDim.x = l.cluster;
        cfg.attrs = l.cluster > 1 ? attr : attr + 1;
        cfg.numAttrs = (l.cluster > 1 ? 1 : 0) + (h->opt_pdl ? 1 : 0);
        GG_CUDA(h, cudaLaunchKernelExC(&cfg, l.fn, l.map ? args : args + 1));
    }
    return GG_OK;
}

}  // namespace gg

namespace {

using gg::fail;
using gg::MoeLaunch;
using gg::refuse;

constexpr int64_t kMaxIndex = int64_t(1) << 31;  // rows and slots are int32 in device memory

bool aligned16(std::initializer_list<const void *> ptrs) {
    uintptr_t all = 0;
    for (const void *p : ptrs)
        all |= reinterpret_cast<uintptr_t>(p);
    return (all & 15u) == 0;
}

bool aligned4(std::initializer_list<const void *> ptrs) {
    uintptr_t all = 0;
    for (const void *p : ptrs)
        all |= reinterpret_cast<uintptr_t>(p);
    return (all & 3u) == 0;
}

// What every prepare call of this file begins with.
int begin(gg_handle *h, const void *p, char *why, size_t why_len) {
    if (!h)
        return GG_ERR_ARG;
    h->ready = false;
    h->moe.launches = 0;
    h->last_error.clear();
    if (why && why_len)
        why[0] = '\0';
    if (!p)
        return fail(h, GG_ERR_ARG, "null problem");
    return GG_OK;
}

// The device's checks and the handle's status word, once the arguments are accepted.
int bind_device(gg_handle *h, gg_stream_t stream, int &num_sms, char *why, size_t why_len) {
    int dev = 0, major = 0, minor = 0;
    GG_CUDA(h, cudaGetDevice(&dev));
    GG_CUDA(h, cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, dev));
    GG_CUDA(h, cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    GG_CUDA(h, cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev));
    if (major != 10 || minor != 0)
        return refuse(h, why, why_len, "needs an sm_100 GPU (B200/GB200)");
    h->device = dev;
    if (!h->d_status)
        GG_CUDA(h, cudaMalloc(&h->d_status, 16));
    GG_CUDA(h, cudaMemsetAsync(h->d_status, 0, 16, stream));
    return GG_OK;
}

int reserve(gg_handle *h, size_t bytes) {
    if (h->ws_cap >= bytes)
        return GG_OK;
    if (h->d_ws)
        cudaFree(h->d_ws);
    h->d_ws = nullptr;
    h->ws_cap = 0;
    GG_CUDA(h, cudaMalloc(&h->d_ws, bytes));
    h->ws_cap = bytes;
    return GG_OK;
}

int reserve_counters(gg_handle *h, size_t bytes, gg_stream_t stream) {
    if (h->counters_cap < bytes) {
        if (h->d_counters)
            cudaFree(h->d_counters);
        h->d_counters = nullptr;
        h->counters_cap = 0;
        GG_CUDA(h, cudaMalloc(&h->d_counters, bytes));
        h->counters_cap = bytes;
    }
    GG_CUDA(h, cudaMemsetAsync(h->d_counters, 0, bytes, stream));
    return GG_OK;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                   const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The handle's tensor map over bytes [depth, rows, cols] in boxes of box_cols (64, with that swizzle) x box_rows.
int encode_bytes_3d(gg_handle *h, const void *base, int64_t cols, int64_t rows, int64_t depth, uint32_t box_cols, uint32_t box_rows) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    GG_CUDA(h, cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !fn)
        return fail(h, GG_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
    const cuuint64_t dim[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(depth)};
    const cuuint64_t stride[2] = {cuuint64_t(cols), cuuint64_t(cols) * cuuint64_t(rows)};
    const cuuint32_t box[3] = {box_cols, box_rows, 1}, estride[3] = {1, 1, 1};
    const CUresult r = reinterpret_cast<EncodeTiledFn>(fn)(
        &h->moe.map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dim, stride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(h, GG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
    return GG_OK;
}

template <class P> void set_params(gg_handle *h, const P &p) {
    static_assert(sizeof(P) <= sizeof(h->moe.params), "parameter block too large");
    std::memcpy(h->moe.params, &p, sizeof(P));
}

int finish(gg_handle *h, gg_stream_t stream, std::initializer_list<MoeLaunch> launches, const char *detail) {
    int n = 0;
    for (const MoeLaunch &l : launches)
        h->moe.launch[n++] = l;
    GG_CUDA(h, cudaStreamSynchronize(stream));  // as gg_prepare: the handle's own buffers are in place
    h->detail = detail;
    h->moe.launches = n;
    h->ready = true;
    return GG_OK;
}

// An entry of the C ABI lets no C++ exception out.
template <class F> int guarded(gg_handle *h, F &&f) noexcept {
    try {
        return f();
    } catch (...) {
        if (h)
            h->ready = false;
        return GG_ERR_ARG;
    }
}

const char *type_name(int t) { return t == GG_F32 ? "fp32" : t == GG_FP16 ? "fp16" : "bf16"; }

// ---- router ----

template <class T, int V> const void *route_fn(bool grad) {
    return grad ? reinterpret_cast<const void *>(&gg::moe::route_grad<T, V>) : reinterpret_cast<const void *>(&gg::moe::route_topk<T, V>);
}
template <class T> const void *route_fn(int experts, bool grad) {
    const int v = (experts + 31) / 32;
    if (v <= 1)
        return route_fn<T, 1>(grad);
    if (v <= 2)
        return route_fn<T, 2>(grad);
    if (v <= 4)
        return route_fn<T, 4>(grad);
    if (v <= 8)
        return route_fn<T, 8>(grad);
    if (v <= 16)
        return route_fn<T, 16>(grad);
    return route_fn<T, 32>(grad);
}
const void *route_fn(int type, int experts, bool grad) {
    return type == GG_F32 ? route_fn<float>(experts, grad)
           : type == GG_FP16 ? route_fn<__half>(experts, grad) : route_fn<__nv_bfloat16>(experts, grad);
}

const char *route_bad(int32_t type, int64_t tokens, int32_t experts, int32_t top_k) {
    if (type != GG_BF16 && type != GG_FP16 && type != GG_F32)
        return "logits_type must be bf16 (0), fp16 (1) or fp32 (2)";
    if (tokens < 0 || tokens >= kMaxIndex)
        return "tokens must be 0..2^31 - 1";
    if (experts < 1 || experts > gg::moe::kMaxExperts)
        return "experts must be 1..1024";
    if (top_k < 1 || top_k > gg::moe::kMaxTopK || top_k > experts)
        return "top_k must be 1..32 and at most experts";
    if (tokens * top_k >= kMaxIndex)
        return "tokens * top_k must be below 2^31";
    return nullptr;
}

// Dynamic shared memory of route_topk: the warps' counters of `experts` experts and lists of top_keys.
size_t route_smem(int warps, int experts) { return size_t(warps) * (size_t(experts) + 128) * 4; }

// How many clusters of route_place the GPU holds at once.
int place_clusters(gg_handle *h, int &fit) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = gg::moe::kPlaceCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(gg::moe::kPlaceCluster, 1, 1);
    cfg.blockDim = dim3(gg::moe::kPlaceThreads, 1, 1);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    GG_CUDA(h, cudaOccupancyMaxActiveClusters(&fit, gg::moe::route_place<gg::moe::kPlaceCluster>, &cfg));
    return GG_OK;
}

int prepare_route(gg_handle *h, const gg_route_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    if (const char *bad = route_bad(q.logits_type, q.tokens, q.experts, q.top_k))
        return refuse(h, why, why_len, bad);
    if (!q.counts || !q.offsets || !q.live || (q.tokens > 0 && (!q.logits || !q.ids || !q.weights || !q.dest || !q.src)))
        return refuse(h, why, why_len, "logits, ids, weights, counts, offsets, live, dest and src must be non-null device pointers");
    if (!aligned16({q.logits}) ||
        !aligned4({q.ids, q.weights, q.lse, q.counts, q.offsets, q.live, q.dest, q.src, q.prob, q.losses}))
        return refuse(h, why, why_len, "logits must be 16-byte aligned, the outputs 4-byte aligned");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    gg::moe::RouteParams p{};
    p.logits = q.logits;
    p.mask = q.mask;
    p.ids = q.ids;
    p.weights = q.weights;
    p.lse = q.lse;
    p.counts = q.counts;
    p.offsets = q.offsets;
    p.live = q.live;
    p.dest = q.dest;
    p.src = q.src;
    p.prob = q.prob;
    p.losses = q.losses;
    p.tokens = q.tokens;
    p.experts = q.experts;
    p.top_k = q.top_k;
    p.normalize = q.normalize != 0;
    p.scale = q.scale;
    // One block where a warp gets two tokens at most and a thread one expert (it finishes alone, in one launch). Else 8 tokens a block,
    // up to 64 as long as that leaves 64 blocks or more, and a block an SM at most: route_place's work grows with the blocks. Us of 256
    // experts and k = 8 with 8 / 16 / 32 / 64 tokens a block: 256 tokens 10.6 / 11.0 / 12.7, 512 12.3 / 11.3 / 12.9, 1000 16.7 / 13.1 / 13.0 /
    // 15.5, 2000 19.0 / 17.5 / 14.9 / 15.6, 4096 20.6 / - / 19.5 / 17.4.
    int v = 1;  // logits a lane: route_fn's V
    while (32 * v < q.experts)
        v *= 2;
    const int warps = gg::moe::route_warps(v);
    const bool alone = q.tokens <= 2 * warps && q.experts <= 32 * warps;
    int64_t each = 8;
    while (each < 64 && (q.tokens + each - 1) / each >= 64)
        each *= 2;
    p.alone = alone;
    p.blocks = alone ? 1 : int(std::max<int64_t>(1, std::min<int64_t>((q.tokens + each - 1) / each, num_sms)));
    // Clusters that share route_place's sums cost their barriers, up to 1.5 us: taken where a thread would load more than 16 rows, with
    // as many blocks as fit at once in clusters (33 of 4; with one more the last runs alone). Us without / with: 16384 tokens of 256 experts
    // 28.4 / 24.3, 8192 22.5 / 18.1, 4096 (64 blocks) 17.5 / 17.9, 16384 of 64 18.8 / 20.1, of 128 21.4 / 20.1, 1000 of 512 16.2 / 13.9, 2000 of
    // 1000 34.6 / 29.0.
    int64_t span = 32;
    while (span < q.experts)
        span *= 2;
    unsigned cluster = 1;
    if (p.blocks * span > 16 * gg::moe::kPlaceThreads) {
        int fit = 0;
        if (const int rc = place_clusters(h, fit))
            return rc;
        if (fit > 0) {
            cluster = gg::moe::kPlaceCluster;
            p.blocks = std::min(p.blocks, int(cluster) * fit - 1);
        }
    }
    p.per_block = std::max<int64_t>(1, (q.tokens + p.blocks - 1) / p.blocks);
    const size_t entries = size_t(p.blocks) * size_t(q.experts + 1);
    if (const int rc = reserve(h, 2 * entries * 4))
        return rc;
    p.block_sums = h->d_ws;
    p.block_counts = reinterpret_cast<int32_t *>(h->d_ws + entries);
    set_params(h, p);
    const void *fn = route_fn(q.logits_type, q.experts, false);
    // The limit belongs to the function, which other handles launch with up to 32 v experts: set for those, never for this problem's.
    GG_CUDA(h, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(route_smem(warps, 32 * v))));
    MoeLaunch topk{fn, unsigned(p.blocks), unsigned(warps) * 32, route_smem(warps, q.experts)};
    MoeLaunch place{cluster > 1 ? reinterpret_cast<const void *>(&gg::moe::route_place<gg::moe::kPlaceCluster>)
                                : reinterpret_cast<const void *>(&gg::moe::route_place<1>),
                    alone ? 0u : (unsigned(p.blocks) / cluster + 1) * cluster, gg::moe::kPlaceThreads, 0};
    place.cluster = cluster;
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_route<%s> experts=%d top_k=%d blocks=%d", type_name(q.logits_type), q.experts, q.top_k, p.blocks);
    return finish(h, stream, {topk, place}, detail);
}

int prepare_route_grad(gg_handle *h, const gg_route_grad_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    if (const char *bad = route_bad(q.logits_type, q.tokens, q.experts, q.top_k))
        return refuse(h, why, why_len, bad);
    if (!q.counts || !q.live || (q.tokens > 0 && (!q.logits || !q.ids || !q.lse || !q.dlogits)))
        return refuse(h, why, why_len, "logits, ids, lse, counts, live and dlogits must be non-null device pointers");
    if (!aligned16({q.logits, q.dlogits}) || !aligned4({q.ids, q.lse, q.counts, q.live, q.dweights, q.dlosses}))
        return refuse(h, why, why_len, "logits and dlogits must be 16-byte aligned, the other operands 4-byte aligned");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    gg::moe::RouteGradParams p{};
    p.logits = q.logits;
    p.mask = q.mask;
    p.ids = q.ids;
    p.lse = q.lse;
    p.counts = q.counts;
    p.live = q.live;
    p.dweights = q.dweights;
    p.dlosses = q.dlosses;
    p.dlogits = q.dlogits;
    p.status = h->d_status;
    p.tokens = q.tokens;
    p.experts = q.experts;
    p.top_k = q.top_k;
    p.normalize = q.normalize != 0;
    p.scale = q.scale;
    set_params(h, p);
    const void *fn = route_fn(q.logits_type, q.experts, true);
    const size_t smem = size_t(gg::moe::kGradWarps) * size_t(q.experts) * 4;
    int per_sm = 0;
    GG_CUDA(h, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, gg::moe::kGradThreads, smem));
    const int64_t blocks = std::min<int64_t>((q.tokens + gg::moe::kGradWarps - 1) / gg::moe::kGradWarps, int64_t(num_sms) * std::max(1, per_sm));
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_route_grad<%s> experts=%d top_k=%d blocks=%d", type_name(q.logits_type), q.experts, q.top_k, int(blocks));
    return finish(h, stream, {MoeLaunch{fn, unsigned(blocks), gg::moe::kGradThreads, smem}}, detail);
}

// ---- dispatch / combine ----

const char *permute_bad(int32_t dtype, int64_t tokens, int32_t top_k, int32_t experts, int64_t hidden) {
    if (dtype != GG_BF16 && dtype != GG_FP16)
        return "dtype must be bf16 (0) or fp16 (1)";
    if (tokens < 0 || tokens >= kMaxIndex)
        return "tokens must be 0..2^31 - 1";
    if (top_k < 1 || top_k > gg::moe::kMaxTopK)
        return "top_k must be 1..32";
    if (experts < 1)
        return "experts must be >= 1";
    if (hidden < 8 || hidden % 8 != 0 || hidden > (int64_t(1) << 30))
        return "hidden must be a multiple of 8 (16-byte rows) in 8..2^30";
    if (tokens * top_k >= kMaxIndex)
        return "tokens * top_k must be below 2^31";
    return nullptr;
}

int prepare_permute(gg_handle *h, const gg_permute_problem &q, int32_t op, gg_stream_t stream, char *why, size_t why_len) {
    if (const char *bad = permute_bad(q.dtype, q.tokens, q.top_k, q.experts, q.hidden))
        return refuse(h, why, why_len, bad);
    gg::moe::PermuteParams p{};
    const bool some = q.tokens > 0;
    if (op == GG_OP_DISPATCH) {
        if (!q.offsets || (some && (!q.x || !q.dest || !q.rows)))
            return refuse(h, why, why_len, "x, dest, offsets and rows must be non-null device pointers");
        p.x = q.x;
        p.out = q.rows;
    } else if (op == GG_OP_COMBINE) {
        if (some && (!q.rows || !q.dest || !q.x))
            return refuse(h, why, why_len, "rows, dest and x must be non-null device pointers");
        p.x = q.rows;
        p.out = q.x;
    } else {
        if (!q.offsets || (some && (!q.dy || !q.dest || !q.drows || (q.dweights && !q.rows))))
            return refuse(h, why, why_len, "dy, rows, dest, offsets and drows must be non-null device pointers");
        p.x = q.rows;
        p.dy = q.dy;
        p.out = q.drows;
        p.dweights = q.dweights;
    }
    if (!aligned16({q.x, q.rows, q.dy, q.drows}) || !aligned4({q.dest, q.offsets, q.weights, q.dweights}))
        return refuse(h, why, why_len, "x, rows, dy and drows must be 16-byte aligned, the other operands 4-byte aligned");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    p.dest = q.dest;
    p.offsets = q.offsets;
    p.weights = q.weights;
    p.status = h->d_status;
    p.rows = q.tokens * q.top_k;
    p.experts = q.experts;
    p.top_k = q.top_k;
    p.vecs = int(q.hidden / 8);
    set_params(h, p);
    const bool half = q.dtype == GG_FP16;
    const void *fn = op == GG_OP_DISPATCH ? reinterpret_cast<const void *>(&gg::moe::dispatch_rows)
                     : op == GG_OP_COMBINE
                         ? (half ? reinterpret_cast<const void *>(&gg::moe::combine_rows<__half>)
                                 : reinterpret_cast<const void *>(&gg::moe::combine_rows<__nv_bfloat16>))
                         : (half ? reinterpret_cast<const void *>(&gg::moe::combine_grad_rows<__half>)
                                 : reinterpret_cast<const void *>(&gg::moe::combine_grad_rows<__nv_bfloat16>));
    // Threads a token, us with at most 128 / 256 / 512 / 1024 of them (launches of a graph): dispatch 16384 x 8 x 7168 356 / 354 / 339 / 330;
    // combine 16384 x 8 x 4096 193 / 196 / 208 / 208, its gradient 7999 x 2 x 2880 39 / 41 / 47 / 47, but combine of 64 tokens x 4 x 7168 17.8 /
    // 11.1 / 6.7 / 4.5. So dispatch takes 1024, the others 128, or as many more as fill the SMs. Then as few vectors a thread as that allows,
    // and no idle warp.
    int most = gg::moe::kPermuteThreads;
    if (op != GG_OP_DISPATCH) {
        most = 128;
        while (most < gg::moe::kPermuteThreads && q.tokens * most < int64_t(num_sms) * 2048)
            most *= 2;
    }
    const int each = (p.vecs + most - 1) / most;
    const unsigned threads = unsigned(((p.vecs + each - 1) / each + 31) / 32 * 32);
    const int64_t blocks = q.tokens;
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_%s<%s> hidden=%lld top_k=%d blocks=%d",
                  op == GG_OP_DISPATCH ? "dispatch" : op == GG_OP_COMBINE ? "combine" : "combine_grad", type_name(q.dtype),
                  static_cast<long long>(q.hidden), q.top_k, int(blocks));
    return finish(h, stream, {MoeLaunch{fn, unsigned(blocks), threads, 0}}, detail);
}

// ---- 4-bit products ----

struct W4Form {
    const void *fn, *gather, *add;
    int tokens;  // of a chunk
    int threads, ctas_per_sm;
    size_t smem;
};
template <class T, int G> W4Form w4_form(bool few, bool zeros) {
    using namespace gg::moe;
    if (few)
        return {zeros ? reinterpret_cast<const void *>(&w4_few<T, G, true>) : reinterpret_cast<const void *>(&w4_few<T, G, false>),
                reinterpret_cast<const void *>(&w4_gather<T, true>), reinterpret_cast<const void *>(&w4_add<T>), kW4FewTokens, kW4FewThreads, 2, kW4FewSmem};
    return {reinterpret_cast<const void *>(&w4_many<T, G>), reinterpret_cast<const void *>(&w4_gather<T, false>), reinterpret_cast<const void *>(&w4_join<T>), W4Many<G>::kTokens,
            kW4ManyThreads, 1, W4Many<G>::kSmemBytes};
}
template <class T> W4Form w4_form(int group, bool few, bool zeros) {
    return group == 32 ? w4_form<T, 32>(few, zeros) : group == 64 ? w4_form<T, 64>(few, zeros) : w4_form<T, 128>(few, zeros);
}

int prepare_w4(gg_handle *h, const gg_w4_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    if (q.dtype != GG_BF16 && q.dtype != GG_FP16)
        return refuse(h, why, why_len, "dtype must be bf16 (0) or fp16 (1)");
    if (q.experts < 1 || q.experts > gg::moe::kW4MaxExperts)
        return refuse(h, why, why_len, "experts must be 1..1024");
    if (q.n < 1 || q.n % 8 != 0 || q.n > (int64_t(1) << 30))
        return refuse(h, why, why_len, "n must be a multiple of 8 (16-byte output row stride) in 8..2^30");
    if (q.k < 1 || q.k % 32 != 0 || q.k > (int64_t(1) << 30))
        return refuse(h, why, why_len, "k must be a multiple of 32 (16-byte stride of 4-bit rows) in 32..2^30");
    if (q.group_size != 32 && q.group_size != 64 && q.group_size != 128)
        return refuse(h, why, why_len, "group_size must be 32, 64 or 128");
    if (q.rows < 0 || q.rows >= kMaxIndex)
        return refuse(h, why, why_len, "rows must be 0..2^31 - 1");
    if (q.src && (q.tokens < 0 || q.tokens >= kMaxIndex || q.top_k < 1 || q.tokens * q.top_k >= kMaxIndex))
        return refuse(h, why, why_len, "with src, tokens must be >= 0, top_k >= 1 and tokens * top_k below 2^31");
    if (!q.offsets || !q.qweight || !q.scales || (q.rows > 0 && (!q.x || !q.out)))
        return refuse(h, why, why_len, "x, qweight, scales, offsets and out must be non-null device pointers");
    if (!aligned16({q.x, q.qweight, q.scales, q.zeros, q.out}) || !aligned4({q.offsets, q.src}))
        return refuse(h, why, why_len, "x, qweight, scales, zeros and out must be 16-byte aligned, offsets and src 4-byte aligned");
    if (q.n * (q.k / 2) >= int64_t(1) << 39)
        return refuse(h, why, why_len, "one expert's weights are too large for a TMA descriptor");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    // Up to a chunk of 8 rows an expert on average, chunks of 8 with mma.sync; above, chunks of up to 32 with tcgen05. Us, few / many. Equal
    // rows an expert (the first form widens the weights a second time from 9 on): 8 experts of 4096 x 7168 in groups of 128, 7 rows 39 / 50, 8
    // 39 / 51, 9 57 / 50; 32 of 7168 x 2048 in groups of 64 with zeros 65 / 96, 65 / 96, 109 / 96; 64 of 4096 x 2048 in groups of 128 59 / 99, 60 /
    // 100, 100 / 99. Uneven rows (up to 3 to 5 times the mean), means of 6, 8, 10, 12, 16: 39 / 50, 48 / 47, 48 / 51, 52 / 51, 65 / 52; 75 / 104,
    // 80 / 108, 95 / 104, 109 / 108, 126 / 118; 69 / 96, 81 / 101, 92 / 102, 99 / 105, 126 / 110.
    const bool few = q.rows <= gg::moe::kW4FewTokens * int64_t(q.experts);
    const W4Form v = q.dtype == GG_FP16 ? w4_form<__half>(q.group_size, few, q.zeros) : w4_form<__nv_bfloat16>(q.group_size, few, q.zeros);
    GG_CUDA(h, cudaFuncSetAttribute(v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(v.smem)));
    if (const int rc = encode_bytes_3d(h, q.qweight, q.k / 2, q.n, q.experts, gg::moe::kW4StepK / 2, gg::moe::kW4TileRows))
        return rc;
    const int ctas = v.ctas_per_sm * num_sms;
    const int blocks = q.rows > 0 ? ctas : 0;
    const int64_t steps = (q.k + gg::moe::kW4StepK - 1) / gg::moe::kW4StepK;
    // partial sums: of the two cut tiles of a CTA, or (few) of the units of split items; a counter: the next unit (few)
    const int64_t tiles = (q.n + gg::moe::kW4TileRows - 1) / gg::moe::kW4TileRows;
    const int64_t items = std::min<int64_t>(q.rows, q.experts + q.rows / v.tokens) * tiles;  // at most
    // Units a CTA and steps a unit, us with 4 of 8 or more / 3 of 8 / 3 of 10 / 3 of 16 / 2 of 16, one token through 8 experts: 4096 x 7168 in
    // groups of 128 36.6 / 36.8 / 37.8 / 38.3 / 38.4, 4096 x 14336 61.8 / 59.7 / 59.4 / 59.5 / 59.1, 4096 x 4096 24.7 / 24.8 / 27.5 / 23.5 / 23.5, 2048 x
    // 2880 15.0 / 15.0 / 16.9 / 20.5 / 20.5; 7168 x 2048 in groups of 64 with zeros 27.6 / 27.6 / 30.5 / 24.3 / 24.3; 1024 x 2048 in groups of 32 14.3
    // / 14.3 / 15.9 / 18.8 / 18.8. So no choice is best throughout.
    int64_t span = steps;
    if (few && items < gg::moe::kW4FewUnits * int64_t(ctas)) {
        const int64_t most = (gg::moe::kW4FewUnits * int64_t(ctas) + items - 1) / std::max<int64_t>(1, items);  // splits
        span = std::max(std::min<int64_t>(8, steps), (steps + most - 1) / most);
    }
    const int64_t splits = (steps + span - 1) / span;
    const size_t sums = size_t(!few ? 2 * ctas : splits > 1 ? items * splits : 0) * size_t(v.tokens) * gg::moe::kW4TileRows * 4;
    if (items > (int64_t(1) << 27))
        return refuse(h, why, why_len, "too many weight rows and experts for one launch");
    if (const int rc = reserve(h, sums + size_t(q.rows + 8 * int64_t(q.experts)) * size_t(steps) * gg::moe::kW4TokenBytes))
        return rc;
    if (const int rc = reserve_counters(h, 4, stream))
        return rc;
    gg::moe::W4Params p{};
    p.x = q.x;
    p.scales = q.scales;
    p.zeros = static_cast<const uint8_t *>(q.zeros);
    const int64_t metas = int64_t(q.experts) * q.n * ((q.k + q.group_size - 1) / q.group_size);
    p.scales_end = static_cast<const uint8_t *>(q.scales) + 2 * metas;  // n is a multiple of 8
    p.zeros_end = static_cast<const uint8_t *>(q.zeros) + metas;
    p.offsets = q.offsets;
    p.src = q.src;
    p.out = q.out;
    p.status = h->d_status;
    p.rows = q.rows;
    p.slots = q.src ? q.tokens * q.top_k : 0;
    p.n = int(q.n);
    p.k = int(q.k);
    p.groups = int((q.k + q.group_size - 1) / q.group_size);
    p.experts = q.experts;
    p.top_k = q.src ? q.top_k : 1;
    p.tiles = int((q.n + gg::moe::kW4TileRows - 1) / gg::moe::kW4TileRows);
    p.steps = int(steps);
    p.chunk = v.tokens;
    p.ctas = ctas;
    p.splits = int(splits);
    p.span = int(span);
    p.ws = h->d_ws;
    p.xs = reinterpret_cast<uint8_t *>(h->d_ws) + sums;
    p.counters = h->d_counters;
    p.timeout_ns = uint64_t(h->opt_timeout_ms) * 1000000u;
    set_params(h, p);
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_w4<%s,%s> n=%lld k=%lld group=%d blocks=%d", type_name(q.dtype), few ? "few" : "many",
                  static_cast<long long>(q.n), static_cast<long long>(q.k), q.group_size, blocks);
    MoeLaunch gather{v.gather, unsigned(std::min<int64_t>(q.rows, 65536)), gg::moe::kW4GatherThreads, 0};
// a block a row, and of few rows one for each 128 pieces
    gather.grid_y = unsigned(std::max<int64_t>(1, std::min<int64_t>((steps * 16 + gg::moe::kW4GatherThreads - 1) / gg::moe::kW4GatherThreads,
                                                                    4 * num_sms / std::max<int64_t>(1, q.rows))));
    MoeLaunch add{v.add, few ? (splits > 1 ? unsigned(std::min<int64_t>(items, 4 * num_sms)) : 0u) : unsigned(blocks), gg::moe::kW4TileRows, 0};
    if (!few)
        add.grid_y = unsigned(v.tokens) / 8;
    return finish(h, stream, {gather, MoeLaunch{v.fn, unsigned(blocks), unsigned(v.threads), v.smem, true}, add}, detail);
}

}  // namespace

extern "C" {

int gg_prepare_route(gg_handle *h, const gg_route_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_route(h, *p, stream, why, why_len);
    });
}

int gg_prepare_route_grad(gg_handle *h, const gg_route_grad_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_route_grad(h, *p, stream, why, why_len);
    });
}

int gg_prepare_permute(gg_handle *h, const gg_permute_problem *p, int32_t op, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        if (op != GG_OP_DISPATCH && op != GG_OP_COMBINE && op != GG_OP_COMBINE_GRAD)
            return fail(h, GG_ERR_ARG, "op must be GG_OP_DISPATCH (3), GG_OP_COMBINE (4) or GG_OP_COMBINE_GRAD (5)");
        return prepare_permute(h, *p, op, stream, why, why_len);
    });
}

int gg_prepare_w4(gg_handle *h, const gg_w4_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_w4(h, *p, stream, why, why_len);
    });
}

}  // extern "C"
