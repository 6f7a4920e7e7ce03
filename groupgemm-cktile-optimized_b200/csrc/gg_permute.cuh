// Tokens into expert order and back: dispatch (one row for each chosen expert), combine (weighted
// sum of a token's rows) and combine's gradients. The gradient of dispatch is combine without weights.
#pragma once

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kPermuteThreads = 1024;  // at most

struct PermuteParams {
    const void *x;           // dispatch: x; combine: rows; combine_grad: rows
    const void *dy;          // combine_grad
    const int32_t *dest;     // [tokens, top_k]
    const int32_t *offsets;  // [experts + 1] (dispatch, combine_grad)
    const float *weights;    // [tokens, top_k] or null = 1
    void *out;               // dispatch: rows; combine: y; combine_grad: drows
    float *dweights;         // combine_grad, or null
    uint32_t *status;
    int64_t rows;
    int experts, top_k;
    int vecs;  // 16-byte vectors a row
};

// A block a token, each thread 16 bytes of its row at a time, and a block of its own for every token: all three are bound by DRAM,
// and it is the many rows in flight that fill it (a warp a token, with four of its rows in flight, took 290 us for combine's
// 16384 x 8 rows of 4096 against 198). The host picks the threads. A thread's loads of dest are one broadcast.
//
// dest's entry of a slot, -1 where it has none (or one that is out of range).
__device__ __forceinline__ int64_t slot_row(const PermuteParams &p, int64_t slot) {
    const int d = p.dest[slot];
    if (d < -1 || d >= p.rows) {
        report(p.status, kSiteSlot);
        return -1;
    }
    return d;
}

// Zeros in the rows past the last expert's end, so that nothing stale is read from them.
__device__ __forceinline__ void zero_tail(const PermuteParams &p) {
    int64_t total = p.offsets[p.experts];
    if (total < 0 || total > p.rows) {
        if (threadIdx.x == 0)
            report(p.status, kSiteOffsets);
        return;
    }
    for (int64_t r = total + blockIdx.x; r < p.rows; r += gridDim.x)
        for (int i = threadIdx.x; i < p.vecs; i += blockDim.x)
            static_cast<uint4 *>(p.out)[r * p.vecs + i] = make_uint4(0, 0, 0, 0);
}

__global__ void __launch_bounds__(kPermuteThreads) dispatch_rows(const PermuteParams p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int64_t t = blockIdx.x;
    for (int i = threadIdx.x; i < p.vecs; i += blockDim.x) {
        const uint4 v = static_cast<const uint4 *>(p.x)[t * p.vecs + i];
        for (int j = 0; j < p.top_k; ++j) {
            const int64_t d = slot_row(p, t * p.top_k + j);
            if (d >= 0)
                static_cast<uint4 *>(p.out)[d * p.vecs + i] = v;
        }
    }
    zero_tail(p);
}

template <class T> __global__ void __launch_bounds__(kPermuteThreads) combine_rows(const PermuteParams p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int64_t t = blockIdx.x;
    for (int i = threadIdx.x; i < p.vecs; i += blockDim.x) {
        float acc[8] = {};
        for (int j = 0; j < p.top_k; ++j) {
            const int64_t d = slot_row(p, t * p.top_k + j);
            if (d < 0)
                continue;
            const float w = p.weights ? p.weights[t * p.top_k + j] : 1.0f;
            const uint4 v = static_cast<const uint4 *>(p.x)[d * p.vecs + i];
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float2 f = unpack2<T>(u[c]);
                acc[2 * c] = fmaf(w, f.x, acc[2 * c]);
                acc[2 * c + 1] = fmaf(w, f.y, acc[2 * c + 1]);
            }
        }
        static_cast<uint4 *>(p.out)[t * p.vecs + i] =
            make_uint4(pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3]), pack2<T>(acc[4], acc[5]), pack2<T>(acc[6], acc[7]));
    }
}

template <class T> __global__ void __launch_bounds__(kPermuteThreads) combine_grad_rows(const PermuteParams p) {
    __shared__ float red[kPermuteThreads / 32];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int64_t t = blockIdx.x;
    for (int j = 0; j < p.top_k; ++j) {
        const int64_t d = slot_row(p, t * p.top_k + j);
        const float w = p.weights ? p.weights[t * p.top_k + j] : 1.0f;
        float dot = 0.0f;
        for (int i = threadIdx.x; d >= 0 && i < p.vecs; i += blockDim.x) {
            const uint4 g = static_cast<const uint4 *>(p.dy)[t * p.vecs + i];
            const uint4 v = p.dweights ? static_cast<const uint4 *>(p.x)[d * p.vecs + i] : make_uint4(0, 0, 0, 0);
            const uint32_t a[4] = {g.x, g.y, g.z, g.w}, b[4] = {v.x, v.y, v.z, v.w};
            uint32_t o[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float2 f = unpack2<T>(a[c]), r = unpack2<T>(b[c]);
                dot = fmaf(f.x, r.x, fmaf(f.y, r.y, dot));
                o[c] = pack2<T>(w * f.x, w * f.y);
            }
            static_cast<uint4 *>(p.out)[d * p.vecs + i] = make_uint4(o[0], o[1], o[2], o[3]);
        }
        if (!p.dweights)
            continue;
        dot = warp_sum(dot);
        if ((threadIdx.x & 31) == 0)
            red[threadIdx.x >> 5] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
            float s = 0.0f;
            for (int w2 = 0; w2 < int(blockDim.x) / 32; ++w2)
                s += red[w2];
            p.dweights[t * p.top_k + j] = d >= 0 ? s : 0.0f;
        }
        __syncthreads();
    }
    zero_tail(p);
}

}  // namespace moe
}  // namespace gg
