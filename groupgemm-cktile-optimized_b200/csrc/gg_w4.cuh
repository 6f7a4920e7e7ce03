// Rows in expert order times their expert's 4-bit weights with group scales, for few rows an expert:
//   out[r, n] = sum over groups g of scale[e, n, g] * sum_{k in g} (q[e, n, k] - zero[e, n, g]) x[row(r), k]
#pragma once

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kW4Warps = 8;
constexpr int kW4Threads = kW4Warps * 32;
constexpr int kW4Rows = 32;    // weight rows (output columns) of a work item
constexpr int kW4Tokens = 32;  // rows of x of a work item
constexpr int kW4MaxExperts = 1024;

struct W4Params {
    const void *x;           // [tokens or rows, k]
    const uint8_t *qweight;  // [experts, n, k / 2], even k in the low four bits
    const void *scales;      // [experts, n, groups]
    const uint8_t *zeros;    // [experts, n, groups] or null = 8
    const int32_t *offsets;  // [experts + 1]
    const int32_t *src;      // [rows] slots, or null: row r reads x[r]
    void *out;               // [rows, n]
    uint32_t *status;
    int64_t rows, slots;  // slots: tokens * top_k
    int n, k, groups, experts, top_k, tiles;
};

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), 16-bit operands.
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four bits as a 16-bit float without a conversion: placed in the low mantissa bits of a power of two
// (1024 in fp16, 128 in bf16) the value is that power + q, exactly; the power + zero is taken away again,
// exactly too (all are integers below 256 resp. 2048).
template <class T> struct W4Magic;
template <> struct W4Magic<__half> {
    static constexpr uint32_t kBias = 0x64006400u;
};
template <> struct W4Magic<__nv_bfloat16> {
    static constexpr uint32_t kBias = 0x43004300u;
};
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b, __half) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
template <class T> __device__ __forceinline__ uint32_t nibbles(uint32_t w, int s, uint32_t bias_zero) {
    return sub2(((w >> (4 * s)) & 0x000f000fu) | W4Magic<T>::kBias, bias_zero, T());
}

// 4 x 4 transpose of words within each quad of lanes: lane t's word c becomes lane c's word t.
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4]) {
    const int t = threadIdx.x & 3;
    {
        const bool odd = t & 1;
        const uint32_t s0 = odd ? w[0] : w[1], s1 = odd ? w[2] : w[3];
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, s0, 1), r1 = __shfl_xor_sync(0xffffffffu, s1, 1);
        if (odd) {
            w[0] = r0;
            w[2] = r1;
        } else {
            w[1] = r0;
            w[3] = r1;
        }
    }
    {
        const bool high = t & 2;
        const uint32_t s0 = high ? w[0] : w[2], s1 = high ? w[1] : w[3];
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, s0, 2), r1 = __shfl_xor_sync(0xffffffffu, s1, 2);
        if (high) {
            w[0] = r0;
            w[1] = r1;
        } else {
            w[2] = r0;
            w[3] = r1;
        }
    }
}

__device__ __forceinline__ uint4 ld_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Sum of one work item: 32 weight rows x up to 8 NT rows of x, over this warp's part of K.
template <class T, int G, int NT>
__device__ __forceinline__ void w4_item(const W4Params &p, int e, int n0, const int32_t *row_of, int c0, int c1, float (&total)[2][NT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const T *x = static_cast<const T *>(p.x);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                total[m][j][i] = 0.0f;
    const T *xrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int r = row_of[8 * j + g];
        xrow[j] = r >= 0 ? x + int64_t(r) * p.k : nullptr;
    }
    for (int c = c0; c < c1; ++c) {
        const int kc = c * 128;
        uint32_t w[2][2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + 16 * m + 8 * h + g;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (n < p.n && kc + 32 * t < p.k)
                    v = ld_stream(p.qweight + ((int64_t(e) * p.n + n) * p.k + kc) / 2 + 16 * t);
                w[m][h][0] = v.x;
                w[m][h][1] = v.y;
                w[m][h][2] = v.z;
                w[m][h][3] = v.w;
                if (G < 128)
                    quad_transpose(w[m][h]);
            }
        constexpr int kParts = 128 / G;  // groups of this stretch of 128
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int group = (kc + part * G) / G;
            if (group >= p.groups)
                break;
            float scale[2][2];
            uint32_t bias[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int n = n0 + 16 * m + 8 * h + g;
                    const int64_t at = (int64_t(e) * p.n + n) * p.groups + group;
                    scale[m][h] = 0.0f;
                    uint32_t z = 8;
                    if (n < p.n) {
                        scale[m][h] = to_f32(static_cast<const T *>(p.scales)[at]);
                        if (p.zeros)
                            z = p.zeros[at] & 15u;
                    }
                    bias[m][h] = W4Magic<T>::kBias + z * 0x00010001u;
                }
            float acc[2][NT][4] = {};
#pragma unroll
            for (int q = 0; q < 4 / kParts; ++q) {
                const int word = part * (4 / kParts) + q;
                const int kx = kc + (G < 128 ? 32 * word + 8 * t : 32 * t + 8 * word);
                uint32_t b[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (xrow[j] && kx < p.k)
                        v = *reinterpret_cast<const uint4 *>(xrow[j] + kx);
                    b[j][0] = __byte_perm(v.x, v.z, 0x5410);  // k, k + 4
                    b[j][1] = __byte_perm(v.x, v.z, 0x7632);  // k + 1, k + 5
                    b[j][2] = __byte_perm(v.y, v.w, 0x5410);
                    b[j][3] = __byte_perm(v.y, v.w, 0x7632);
                }
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int s = 0; s < 4; s += 2) {
                        const uint32_t a0 = nibbles<T>(w[m][0][word], s, bias[m][0]), a1 = nibbles<T>(w[m][1][word], s, bias[m][1]);
                        const uint32_t a2 = nibbles<T>(w[m][0][word], s + 1, bias[m][0]), a3 = nibbles<T>(w[m][1][word], s + 1, bias[m][1]);
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            mma16816<T>(acc[m][j], a0, a1, a2, a3, b[j][s], b[j][s + 1]);
                    }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        total[m][j][i] = fmaf(scale[m][i >> 1], acc[m][j][i], total[m][j][i]);
        }
    }
}

template <class T, int G, int NT>
__device__ __forceinline__ void w4_run(const W4Params &p, int e, int n0, const int32_t *row_of, int r0, int count, float *sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int chunks = (p.k + 127) / 128, per = (chunks + kW4Warps - 1) / kW4Warps;
    float total[2][NT][4];
    w4_item<T, G, NT>(p, e, n0, row_of, min(chunks, warp * per), min(chunks, (warp + 1) * per), total);
    // the warps' sums, [warp][row of x][weight row]
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums[(warp * 8 * NT + 8 * j + 2 * t + (i & 1)) * kW4Rows + 16 * m + 8 * (i >> 1) + g] = total[m][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < count * kW4Rows; i += kW4Threads) {
        const int r = i / kW4Rows, c = i % kW4Rows;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kW4Warps; ++w)
            s += sums[(w * 8 * NT + r) * kW4Rows + c];
        if (n0 + c < p.n)
            static_cast<T *>(p.out)[int64_t(r0 + r) * p.n + n0 + c] = from_f32<T>(s);
    }
    __syncthreads();
}

template <class T, int G> __global__ void __launch_bounds__(kW4Threads) w4_rows(const W4Params p) {
    __shared__ int start[kW4MaxExperts + 1];  // first row of each expert, checked
    __shared__ int first[kW4MaxExperts + 1];  // row chunks of the experts before
    __shared__ int32_t row_of[kW4Tokens];
    __shared__ float sums[kW4Warps * kW4Tokens * kW4Rows];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int E = p.experts, tid = threadIdx.x;
    // offsets come from the device: each is held to the range the rows allow
    for (int e = tid; e <= E; e += kW4Threads) {
        const int64_t v = p.offsets[e];
        const int64_t before = e ? p.offsets[e - 1] : 0;
        if (v < before || v > p.rows || before < 0)
            report(p.status, kSiteOffsets);
        start[e] = int(max(int64_t(0), min(v, p.rows)));
    }
    __syncthreads();
    {
        const int per = (E + kW4Threads - 1) / kW4Threads;
        int sum = 0;
        for (int i = 0; i < per; ++i) {
            const int e = tid * per + i;
            if (e < E)
                sum += (max(0, start[e + 1] - start[e]) + kW4Tokens - 1) / kW4Tokens;
        }
        int total, at = block_scan(sum, total);
        for (int i = 0; i < per; ++i) {
            const int e = tid * per + i;
            if (e < E) {
                first[e] = at;
                at += (max(0, start[e + 1] - start[e]) + kW4Tokens - 1) / kW4Tokens;
            }
        }
        if (tid == 0)
            first[E] = total;
        __syncthreads();
    }
    const int64_t items = int64_t(first[E]) * p.tiles;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        // the item's expert: the last one whose first chunk's items start at or before it
        int lo = 0, hi = E - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (int64_t(first[mid]) * p.tiles <= item)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int e = lo;
        const int chunks = first[e + 1] - first[e];
        const int64_t at = item - int64_t(first[e]) * p.tiles;
        const int tile = int(at / chunks), chunk = int(at % chunks);
        const int r0 = start[e] + chunk * kW4Tokens, count = min(kW4Tokens, start[e + 1] - r0);
        if (tid < kW4Tokens) {
            int64_t r = -1;
            if (tid < count) {
                r = r0 + tid;
                if (p.src) {
                    const int s = p.src[r];
                    if (s < 0 || s >= p.slots) {
                        report(p.status, kSiteSrc);
                        r = -1;
                    } else {
                        r = s / p.top_k;
                    }
                }
            }
            row_of[tid] = int(r);
        }
        __syncthreads();
        if (count <= 8)
            w4_run<T, G, 1>(p, e, tile * kW4Rows, row_of, r0, count, sums);
        else if (count <= 16)
            w4_run<T, G, 2>(p, e, tile * kW4Rows, row_of, r0, count, sums);
        else
            w4_run<T, G, 4>(p, e, tile * kW4Rows, row_of, r0, count, sums);
    }
    // rows of no expert are zero
    const int64_t head = start[0], tail = start[E];
    const int64_t none = head + (p.rows - tail);
    for (int64_t i = blockIdx.x; i < none; i += gridDim.x) {
        const int64_t r = i < head ? i : tail + (i - head);
        for (int c = tid; c < p.n; c += kW4Threads)
            static_cast<T *>(p.out)[r * p.n + c] = from_f32<T>(0.0f);
    }
}

}  // namespace moe
}  // namespace gg
