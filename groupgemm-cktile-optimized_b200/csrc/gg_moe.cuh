// What the kernels of the layer operators share (gg_route.cuh, gg_permute.cuh, gg_w4.cuh, gg_norm.cuh,
// gg_i8.cuh): element conversions, warp reductions and the status word's index checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "gg_kernel.cuh"
#include "gg_ptx.cuh"

namespace gg {
namespace moe {

// Each kernel starts while the one before it in the stream ends. What that one may still write (rows, scales, statistics, offsets) is read after
// the kernel's wait and never by the read-only path (__ldg, ld.global.nc), which asks that it be unchanged for the whole of the kernel's life.

// Sites of the index checks (status word kStatusBounds | site): these indices come from device
// memory that the host never sees, so a kernel checks each before it uses it as an address; one
// that is out of range is recorded (the first wins) and its access skipped.
enum Site : uint32_t {
    kSiteSlot = 0x10,     // dest entry neither -1 nor a row
    kSiteSrc = 0x11,      // src entry not a slot
    kSiteOffsets = 0x12,  // offsets falling, or past the rows
    kSiteExpert = 0x13,   // ids entry neither -1 nor an expert
};

__device__ __forceinline__ void report(uint32_t *status, Site site) { atomicCAS(status, 0u, kStatusBounds | site); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The two 16-bit values of a 32-bit word, and back (round to nearest even).
template <class T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Tensor Memory: 32 lanes x 16 columns, and the wait that its uses are tied to.
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32"
                 " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// Exclusive prefix sum of v over the block's threads; total: the whole sum.
__device__ __forceinline__ int block_scan(int v, int &total) {
    __shared__ int part[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o)
            s += u;
    }
    if (lane == 31)
        part[warp] = s;
    __syncthreads();
    if (warp == 0) {
        int q = lane < warps ? part[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o)
                q += u;
        }
        part[lane] = q;
    }
    __syncthreads();
    total = part[warps - 1];
    const int before = warp ? part[warp - 1] : 0;
    __syncthreads();
    return before + s - v;
}

}  // namespace moe
}  // namespace gg
