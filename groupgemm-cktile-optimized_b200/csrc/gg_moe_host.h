// What the prepare calls of the layer operators share (gg_moe.cu, gg_norm_i8.cu): argument checks, the handle's buffers, tensor
// maps and the launch plan.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "gg_b200.h"
#include "gg_handle.h"

namespace gg {
namespace host {

constexpr int64_t kMaxIndex = int64_t(1) << 31;  // rows and slots are int32 in device memory

inline bool aligned16(std::initializer_list<const void *> ptrs) {
    uintptr_t all = 0;
    for (const void *p : ptrs)
        all |= reinterpret_cast<uintptr_t>(p);
    return (all & 15u) == 0;
}

inline bool aligned4(std::initializer_list<const void *> ptrs) {
    uintptr_t all = 0;
    for (const void *p : ptrs)
        all |= reinterpret_cast<uintptr_t>(p);
    return (all & 3u) == 0;
}

// What every prepare call of this file begins with.
inline int begin(gg_handle *h, const void *p, char *why, size_t why_len) {
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
inline int bind_device(gg_handle *h, gg_stream_t stream, int &num_sms, char *why, size_t why_len) {
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

inline int reserve(gg_handle *h, size_t bytes) {
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

inline int reserve_counters(gg_handle *h, size_t bytes, gg_stream_t stream) {
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

// A tensor map over bytes: boxes of box_cols (a row of the swizzle) x box_rows.
inline int encode_bytes(gg_handle *h, CUtensorMap &map, const void *base, unsigned rank, const cuuint64_t *dim, const cuuint64_t *stride,
                        const cuuint32_t *box, CUtensorMapSwizzle swizzle) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    GG_CUDA(h, cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !fn)
        return fail(h, GG_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
    const cuuint32_t estride[3] = {1, 1, 1};
    const CUresult r = reinterpret_cast<EncodeTiledFn>(fn)(
        &map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void *>(base), dim, stride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(h, GG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
    return GG_OK;
}
// Over [depth, rows, cols].
inline int encode_bytes_3d(gg_handle *h, CUtensorMap &map, const void *base, int64_t cols, int64_t rows, int64_t depth, uint32_t box_cols,
                           uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    const cuuint64_t dim[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(depth)};
    const cuuint64_t stride[2] = {cuuint64_t(cols), cuuint64_t(cols) * cuuint64_t(rows)};
    const cuuint32_t box[3] = {box_cols, box_rows, 1};
    return encode_bytes(h, map, base, 3, dim, stride, box, swizzle);
}
// Over [rows, cols].
inline int encode_bytes_2d(gg_handle *h, CUtensorMap &map, const void *base, int64_t cols, int64_t rows, uint32_t box_cols, uint32_t box_rows,
                           CUtensorMapSwizzle swizzle) {
    const cuuint64_t dim[2] = {cuuint64_t(cols), cuuint64_t(rows)}, stride[1] = {cuuint64_t(cols)};
    const cuuint32_t box[2] = {box_cols, box_rows};
    return encode_bytes(h, map, base, 2, dim, stride, box, swizzle);
}

template <class P> void set_params(gg_handle *h, const P &p) {
    static_assert(sizeof(P) <= sizeof(h->moe.params), "parameter block too large");
    std::memcpy(h->moe.params, &p, sizeof(P));
}

inline int finish(gg_handle *h, gg_stream_t stream, std::initializer_list<MoeLaunch> launches, const char *detail) {
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

inline const char *type_name(int t) { return t == GG_F32 ? "fp32" : t == GG_FP16 ? "fp16" : "bf16"; }

}  // namespace host
}  // namespace gg
