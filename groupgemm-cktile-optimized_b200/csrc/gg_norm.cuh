// Layer norm of each token and its gradients, and the rounding of rows to 8-bit integers.
//   s = x + residual (rounded to the type)   m = mean s   r = 1 / sqrt(mean (s - m)^2 + eps)   y = (s - m) r gamma + beta
//   ds = r (d - mean d - c mean(d c)) + dsum   with c = (s - m) r, d = dy gamma;   dgamma = sum_t dy c, dbeta = sum_t dy
//
// What bounds them: each row is read once and written once. One block an SM stays for the whole launch; its warps form
// groups that take a row each, a vector of 8 values or two a thread, held in registers between the sums and the result. Rows come through a
// ring in shared memory, bulk copies a few rows ahead, so that the sums' latency (shuffles and a barrier a row) passes while
// the next rows are on their way, and a thread's weight, bias and sums of gradients stay in registers from row to row.
#pragma once

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kNormMaxHidden = 16384;
constexpr int kNormSmem = 200 * 1024;  // of a block's ring
constexpr int kNormMaxSlots = 8;       // rows that a group's ring holds
constexpr int kNormMaxGroups = 15;     // each has a named barrier beside the block's own

struct NormParams {
    const void *x, *residual;   // [rows, hidden]
    const void *gamma, *beta;   // [hidden] or null = 1, 0
    void *sum, *y;              // [rows, hidden] or null
    float *mean, *rstd;         // [rows] or null
    int8_t *q;                  // [rows, hidden] or null
    float *q_scales;            // [rows]
    uint32_t *status;           // [0] status word, [2] timeouts of this launch
    int64_t rows;
    int vecs;                   // 8 values each, of a row
    int warps, groups, slots;   // a group's warps, a block's groups, a ring's rows
    float eps;
    uint64_t timeout_ns;
};

struct NormGradParams {
    const void *x, *dy, *dsum;  // [rows, hidden]; dsum may be null
    const void *gamma;          // [hidden] or null = 1
    const float *mean, *rstd;   // [rows]
    void *dx;                   // [rows, hidden]
    float *dgamma, *dbeta;      // [hidden] or null
    float *parts;               // [blocks, 2, hidden]
    uint32_t *status;
    int64_t rows;
    int vecs;
    int warps, groups, slots;
    int blocks;
    uint64_t timeout_ns;
};

// Untiled bulk copy global -> shared, 16-byte aligned on both sides, a multiple of 16 bytes.
__device__ __forceinline__ void row_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint4 lds_row(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Eight values of a row in the words that hold them.
template <class T> struct Vec8 {
    uint4 w;
    __device__ __forceinline__ void lds(uint32_t row, int vec) { w = lds_row(row + uint32_t(vec) * 16u); }
    __device__ __forceinline__ void ldg(const void *row, int vec) { w = __ldg(static_cast<const uint4 *>(row) + vec); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y), c = unpack2<T>(w.z), d = unpack2<T>(w.w);
        f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        w = make_uint4(moe::pack2<T>(f[0], f[1]), moe::pack2<T>(f[2], f[3]), moe::pack2<T>(f[4], f[5]), moe::pack2<T>(f[6], f[7]));
    }
    __device__ __forceinline__ void stg(void *row, int vec) const { __stcs(static_cast<uint4 *>(row) + vec, w); }
    // The largest magnitude's bits (NaN above all), of two columns at a time; bits(): as fp32's.
    __device__ __forceinline__ uint32_t top(uint32_t so_far) const {
        return __vimax3_s16x2(__vimax3_s16x2(so_far, w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), w.z & 0x7fff7fffu, w.w & 0x7fff7fffu);
    }
    static __device__ __forceinline__ uint32_t bits(uint32_t top) {
        const float2 v = unpack2<T>(max(top & 0xffffu, top >> 16));
        return __float_as_uint(v.x);
    }
};
template <> struct Vec8<float> {
    float4 a, b;
    __device__ __forceinline__ void lds(uint32_t row, int vec) {
        const uint4 u = lds_row(row + uint32_t(vec) * 32u), v = lds_row(row + uint32_t(vec) * 32u + 16u);
        a = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        b = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ __forceinline__ void ldg(const void *row, int vec) {
        a = __ldg(static_cast<const float4 *>(row) + 2 * vec);
        b = __ldg(static_cast<const float4 *>(row) + 2 * vec + 1);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        a = make_float4(f[0], f[1], f[2], f[3]);
        b = make_float4(f[4], f[5], f[6], f[7]);
    }
    __device__ __forceinline__ void stg(void *row, int vec) const {
        __stcs(static_cast<float4 *>(row) + 2 * vec, a);
        __stcs(static_cast<float4 *>(row) + 2 * vec + 1, b);
    }
    __device__ __forceinline__ uint32_t top(uint32_t so_far) const {
        const uint32_t m = 0x7fffffffu;
        return max(max(max(__float_as_uint(a.x) & m, __float_as_uint(a.y) & m), max(__float_as_uint(a.z) & m, __float_as_uint(a.w) & m)),
                   max(max(max(__float_as_uint(b.x) & m, __float_as_uint(b.y) & m), max(__float_as_uint(b.z) & m, __float_as_uint(b.w) & m)), so_far));
    }
    static __device__ __forceinline__ uint32_t bits(uint32_t top) { return top; }
};

// ---- rounding to 8-bit integers ----
//
// scale = top / 127 and q = the whole number nearest to 127 v / top, halves to the even one, for the row's largest magnitude top: of
// the exact quotient, so that the result does not depend on how it is computed. v (127 / top) is off by at most 127 * 2^-24 = 7.6e-6 by
// the division's rounding, and the sum with 1.5 * 2^23 that brings its nearest whole number into the low bits rounds once. Where
// that leaves the choice open for one of eight values (within 2e-5 of a half), all eight are decided exactly, by the sign of
// 254 v - (2 f + 1) top, f = floor: both products are split into a rounded part and its error by fma, and their difference is exact (it is small).
// So are rows whose top is below 2^-60 or above 2^60, scaled by 2^80 or 2^-80 first so that nothing here leaves fp32's normal range.
// A row of zeros has scale 0 and q 0; one that holds NaN or an infinity has scale NaN and q 0.
// (Each value by itself, with a conversion and the test for a half: 32768 rows of 7168 in 230 us in place of the bytes' 108.)
struct Rounding {
    float top, inverse, up;
    bool zero, careful;  // all q are 0; all values the exact way
    __device__ __forceinline__ Rounding(uint32_t top_bits, float &scale) {  // of the largest magnitude's bits (NaN above all)
        top = __uint_as_float(top_bits);
        const bool odd = top_bits >= 0x7f800000u;
        scale = odd ? __uint_as_float(0x7fc00000u) : __fdiv_rn(top, 127.0f);
        zero = odd || top_bits == 0u;
        up = top < 8.6736174e-19f ? 1.2089258e24f : top > 1.1529215e18f ? 8.2718061e-25f : 1.0f;  // 2^-60, 2^80; 2^60, 2^-80
        careful = zero || up != 1.0f;
        top = zero ? 1.0f : top * up;
        inverse = __fdiv_rn(127.0f, top);
    }
    __device__ __forceinline__ uint32_t exact(float v) const {
        if (zero)
            return 0u;
        const float a = fabsf(v) * up, t = a * inverse;
        float m = rintf(t);
        if (fabsf(t - m) > 0.49998f) {
            const float f = floorf(t), b = 2.0f * f + 1.0f, p = b * top;
            const float e = fmaf(b, top, -p), r = fmaf(254.0f, a, -p);
            m = r > e ? f + 1.0f : r < e ? f : 2.0f * rintf(0.5f * (f + 0.5f));
        }
        return uint32_t(v < 0.0f ? -int(m) : int(m));
    }
    __device__ __forceinline__ uint2 operator()(const float (&v)[8]) const {
        uint32_t n[8];
        float worst = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = fmaf(v[i], inverse, 12582912.0f);  // its low byte is the number's
            worst = fmaxf(worst, fabsf(fmaf(v[i], inverse, 12582912.0f - s)));
            n[i] = __float_as_uint(s);
        }
        if (worst > 0.49998f || careful)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                n[i] = exact(v[i]);
        return make_uint2(__byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410),
                          __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410));
    }
};

struct QuantParams {
    const void *x;    // [rows, k]
    int8_t *q;        // [rows, k]
    float *scales;    // [rows]
    int64_t rows;
    int vecs;         // k / 8
};

// One row by a block: up to kQuantHeld vectors a thread stay in registers between the largest magnitude and the rounding, what is
// longer is read again. part: 16 words of shared memory, other ones for the next row.
constexpr int kQuantHeld = 4;
template <class T> __device__ __forceinline__ void quant_row(const void *row, int8_t *to, float *scale_to, int vecs, uint32_t *part) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    Vec8<T> v[kQuantHeld];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i) {
        const int at = tid + i * int(blockDim.x);
        if (at < vecs)
            v[i].ldg(row, at);
    }
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i)
        if (tid + i * int(blockDim.x) < vecs)
            top = v[i].top(top);
    for (int at = tid + kQuantHeld * int(blockDim.x); at < vecs; at += blockDim.x) {
        Vec8<T> u;
        u.ldg(row, at);
        top = u.top(top);
    }
    top = __reduce_max_sync(0xffffffffu, Vec8<T>::bits(top));
    if (lane == 0)
        part[warp] = top;
    __syncthreads();  // a warp writes these words again only after the next row's barrier
    top = __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
    float scale;
    const Rounding by(top, scale);
    if (tid == 0)
        *scale_to = scale;
    uint2 *q = reinterpret_cast<uint2 *>(to);
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i) {
        const int at = tid + i * int(blockDim.x);
        if (at < vecs) {
            float f[8];
            v[i].get(f);
            q[at] = by(f);
        }
    }
    for (int at = tid + kQuantHeld * int(blockDim.x); at < vecs; at += blockDim.x) {
        Vec8<T> u;
        float f[8];
        u.ldg(row, at);
        u.get(f);
        q[at] = by(f);
    }
}

// A block a row (and every gridDim.x-th after it).
template <class T> __global__ void __launch_bounds__(512) quant_rows(const __grid_constant__ QuantParams p) {
    __shared__ uint32_t part[2][16];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    int turn = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1)
        quant_row<T>(static_cast<const uint8_t *>(p.x) + r * p.vecs * int64_t(8 * sizeof(T)), p.q + r * p.vecs * 8, p.scales + r, p.vecs, part[turn]);
}

// ---- rows through a ring in shared memory ----

// A group of warps of a block, its ring of rows and its barrier. All threads of a group take the same steps; a wait that gives up is
// recorded and the group goes on without waiting or storing, so that its barriers stay matched.
template <int kTensors> struct RowRing {
    uint32_t base, bars;
    uint32_t row_bytes;
    int tensors;                     // that are there: the first ones of `from`
    int slots, group, threads, tid;  // tid within the group
    int64_t first, stride, rows;
    const uint8_t *from[kTensors];
    Abort ab;
    bool ok = true;

    __device__ __forceinline__ uint32_t at(int slot, int tensor) const { return base + uint32_t(slot * tensors + tensor) * row_bytes; }
    __device__ __forceinline__ void sync() const {
        if (threads == 32)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
    }
    // By one thread, when all have read the slot.
    __device__ __forceinline__ void load(int slot, int64_t row) const {
        if (tid != 0 || row >= rows || !ok)
            return;
        ptx::mbar_arrive_expect_tx(bars + 8u * slot, uint32_t(tensors) * row_bytes, 1u);
#pragma unroll
        for (int t = 0; t < kTensors; ++t)
            if (t < tensors)
                row_load(at(slot, t), from[t] + row * row_bytes, row_bytes, bars + 8u * slot);
    }
    __device__ __forceinline__ void wait(int slot, uint32_t phase) {
        if (ok)
            ok = wait_all(bars + 8u * slot, phase, ab, kStatusTimeout | kRoleProducer | uint32_t(slot));
    }
};

// Sets up a block's rings; by all threads, which are together after it.
template <int kTensors, class P>
__device__ __forceinline__ RowRing<kTensors> row_ring(const P &p, int tensors, uint32_t smem, uint64_t *bars, volatile uint32_t *flag, int row_bytes) {
    RowRing<kTensors> g;
    g.threads = p.warps * 32;
    g.group = int(threadIdx.x) / g.threads;
    g.tid = int(threadIdx.x) - g.group * g.threads;
    g.tensors = tensors;
    g.slots = p.slots;
    g.row_bytes = uint32_t(row_bytes);
    g.base = smem + uint32_t(g.group * p.slots * tensors) * g.row_bytes;
    g.bars = ptx::smem_addr(bars + g.group * kNormMaxSlots);
    g.first = int64_t(blockIdx.x) * p.groups + g.group;
    g.stride = int64_t(gridDim.x) * p.groups;
    g.rows = p.rows;
    g.ab = Abort{p.status + 2, flag, p.timeout_ns};
    if (g.tid == 0)
        for (int s = 0; s < p.slots; ++s)
            ptx::mbar_init(g.bars + 8u * s, 1);
    if (threadIdx.x == 0)
        *flag = 0u;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    __syncthreads();
    ptx::griddep_wait();
    ptx::fence_proxy_async_global();
    ptx::griddep_launch_dependents();
    return g;
}

// After a block's last row: what a wait reported goes to the status word.
__device__ __forceinline__ void row_ring_end(uint32_t *status, volatile uint32_t *flag) {
    __syncthreads();
    if (*flag != 0u) {
        // let copies already issued drain before the memory they target goes away
        const uint64_t t0 = ptx::globaltimer();
        while (ptx::globaltimer() - t0 < 200000ull)
            __nanosleep(1000);
        if (threadIdx.x == 0)
            atomicCAS(status, 0u, *reinterpret_cast<volatile uint32_t *>(status + 2));
    }
}

// Mean and variance without cancellation: each warp its own mean and the squares around it, joined by
//   sum (v - m)^2 = sum over warps of (squares_w + n_w (m_w - m)^2).
template <class T, class W, int V, int kMax>
__global__ void __launch_bounds__(kMax, 1) norm_rows(const __grid_constant__ NormParams p) {
    extern __shared__ __align__(1024) uint8_t norm_smem[];
    __shared__ uint64_t bars[kNormMaxGroups * kNormMaxSlots];
    __shared__ float2 part[kNormMaxGroups * 2 * 32];
    __shared__ uint32_t tops[kNormMaxGroups * 2 * 32];
    __shared__ volatile uint32_t flag;
    RowRing<2> g = row_ring<2>(p, p.residual ? 2 : 1, ptx::smem_addr(norm_smem), bars, &flag, p.vecs * int(8 * sizeof(T)));
    g.from[0] = static_cast<const uint8_t *>(p.x);
    g.from[1] = static_cast<const uint8_t *>(p.residual);
    const int warp = g.tid >> 5, lane = g.tid & 31;
    for (int s = 0; s < g.slots; ++s)
        g.load(s, g.first + s * g.stride);
    // values of warp w (and of this one)
    auto count = [&](int w) {
        int n = 0;
#pragma unroll
        for (int v = 0; v < V; ++v)
            n += min(32, max(0, p.vecs - v * g.threads - w * 32));
        return float(8 * n);
    };
    const float mine = count(warp), inv_mine = mine > 0.0f ? 1.0f / mine : 0.0f;
    const float theirs = lane < p.warps ? count(lane) : 0.0f, inv_theirs = theirs > 0.0f ? 1.0f / theirs : 0.0f;
    const float inv_hidden = 1.0f / float(8 * p.vecs);
    Vec8<W> gamma[V], beta[V];
    {
        const float one[8] = {1, 1, 1, 1, 1, 1, 1, 1}, none[8] = {};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            gamma[v].set(one);
            beta[v].set(none);
            if (p.gamma && at < p.vecs)
                gamma[v].ldg(p.gamma, at);
            if (p.beta && at < p.vecs)
                beta[v].ldg(p.beta, at);
        }
    }
    int slot = 0, turn = 0;
    uint32_t phase = 0;
    for (int64_t r = g.first; r < p.rows; r += g.stride) {
        g.wait(slot, phase);
        const int64_t row = r * p.vecs;  // in vectors
        float f[V][8];
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (at < p.vecs) {
                Vec8<T> x;
                x.lds(g.at(slot, 0), at);
                x.get(f[v]);
                if (p.residual) {
                    float a[8];
                    x.lds(g.at(slot, 1), at);
                    x.get(a);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        f[v][i] += a[i];
                    x.set(f[v]);
                    x.get(f[v]);
                    if (p.sum && g.ok)
                        x.stg(static_cast<uint8_t *>(p.sum) + row * int64_t(8 * sizeof(T)), at);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sum += f[v][i];
            }
        }
        sum = warp_sum(sum);
        float squares = 0.0f;
        const float m_warp = sum * inv_mine;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (g.tid + v * g.threads < p.vecs)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    squares = fmaf(f[v][i] - m_warp, f[v][i] - m_warp, squares);
        squares = warp_sum(squares);
        float2 *mailbox = part + (g.group * 2 + turn) * 32;
        if (lane == 0)
            mailbox[warp] = make_float2(sum, squares);
        g.sync();  // the slot has been read, too
        g.load(slot, r + g.slots * g.stride);
        const float2 w = lane < p.warps ? mailbox[lane] : make_float2(0.0f, 0.0f);
        const float mean = warp_sum(w.x) * inv_hidden;
        const float off = w.x * inv_theirs - mean;
        const float var = warp_sum(fmaf(theirs * off, off, w.y)) * inv_hidden;
        const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(var + p.eps));
        if (g.tid == 0 && g.ok) {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
        uint32_t top = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (at < p.vecs) {
                float a[8], b[8];
                gamma[v].get(a);
                beta[v].get(b);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    f[v][i] = fmaf((f[v][i] - mean) * rstd, a[i], b[i]);
                Vec8<T> y;
                y.set(f[v]);
                if (p.y && g.ok)
                    y.stg(static_cast<uint8_t *>(p.y) + row * int64_t(8 * sizeof(T)), at);
                if (p.q) {
                    top = y.top(top);
                    y.get(f[v]);  // the integers are of y as it is written
                }
            }
        }
        if (p.q) {
            uint32_t *box = tops + (g.group * 2 + turn) * 32;
            top = __reduce_max_sync(0xffffffffu, Vec8<T>::bits(top));
            if (lane == 0)
                box[warp] = top;
            g.sync();
            top = __reduce_max_sync(0xffffffffu, lane < p.warps ? box[lane] : 0u);
            float scale;
            const Rounding by(top, scale);
            if (g.tid == 0 && g.ok)
                p.q_scales[r] = scale;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int at = g.tid + v * g.threads;
                if (at < p.vecs && g.ok)
                    reinterpret_cast<uint2 *>(p.q)[row + at] = by(f[v]);
            }
        }
        turn ^= 1;
        if (++slot == g.slots) {
            slot = 0;
            phase ^= 1u;
        }
    }
    row_ring_end(p.status, &flag);
}

// The gradients: a block's sums of dgamma and dbeta stay in registers over its rows, its groups' are added in order, and each block
// leaves its sums for norm_grad_sum.
template <class T, class W, int V, int kMax>
__global__ void __launch_bounds__(kMax, 1) norm_grad_rows(const __grid_constant__ NormGradParams p) {
    extern __shared__ __align__(1024) uint8_t norm_smem[];
    __shared__ uint64_t bars[kNormMaxGroups * kNormMaxSlots];
    __shared__ float2 part[kNormMaxGroups * 2 * 32];
    __shared__ volatile uint32_t flag;
    RowRing<3> g = row_ring<3>(p, p.dsum ? 3 : 2, ptx::smem_addr(norm_smem), bars, &flag, p.vecs * int(8 * sizeof(T)));
    g.from[0] = static_cast<const uint8_t *>(p.x);
    g.from[1] = static_cast<const uint8_t *>(p.dy);
    g.from[2] = static_cast<const uint8_t *>(p.dsum);
    const int warp = g.tid >> 5, lane = g.tid & 31;
    for (int s = 0; s < g.slots; ++s)
        g.load(s, g.first + s * g.stride);
    const float inv_hidden = 1.0f / float(8 * p.vecs);
    Vec8<W> gamma[V];
    float dgamma[V][8] = {}, dbeta[V][8] = {};
    {
        const float one[8] = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            gamma[v].set(one);
            if (p.gamma && g.tid + v * g.threads < p.vecs)
                gamma[v].ldg(p.gamma, g.tid + v * g.threads);
        }
    }
    float mean = 0.0f, rstd = 0.0f;
    if (g.first < p.rows) {
        mean = __ldg(p.mean + g.first);
        rstd = __ldg(p.rstd + g.first);
    }
    int slot = 0, turn = 0;
    uint32_t phase = 0;
    for (int64_t r = g.first; r < p.rows; r += g.stride) {
        float next_mean = 0.0f, next_rstd = 0.0f;
        if (r + g.stride < p.rows) {
            next_mean = __ldg(p.mean + r + g.stride);
            next_rstd = __ldg(p.rstd + r + g.stride);
        }
        g.wait(slot, phase);
        Vec8<T> x[V], dy[V], more[V];
        float along = 0.0f, level = 0.0f;  // sums of d c and of d
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (at < p.vecs) {
                x[v].lds(g.at(slot, 0), at);
                dy[v].lds(g.at(slot, 1), at);
                if (p.dsum)
                    more[v].lds(g.at(slot, 2), at);
                float a[8], b[8], w[8];
                x[v].get(a);
                dy[v].get(b);
                gamma[v].get(w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float c = (a[i] - mean) * rstd, d = b[i] * w[i];
                    level += d;
                    along = fmaf(d, c, along);
                    dgamma[v][i] = fmaf(b[i], c, dgamma[v][i]);
                    dbeta[v][i] += b[i];
                }
            }
        }
        along = warp_sum(along);
        level = warp_sum(level);
        float2 *mailbox = part + (g.group * 2 + turn) * 32;
        if (lane == 0)
            mailbox[warp] = make_float2(along, level);
        g.sync();  // the slot has been read, too
        g.load(slot, r + g.slots * g.stride);
        const float2 s = lane < p.warps ? mailbox[lane] : make_float2(0.0f, 0.0f);
        along = warp_sum(s.x) * inv_hidden;
        level = warp_sum(s.y) * inv_hidden;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (at < p.vecs) {
                float a[8], b[8], w[8];
                x[v].get(a);
                dy[v].get(b);
                gamma[v].get(w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float c = (a[i] - mean) * rstd;
                    a[i] = rstd * (fmaf(b[i], w[i], -level) - c * along);
                }
                if (p.dsum) {
                    more[v].get(b);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        a[i] += b[i];
                }
                x[v].set(a);
                if (g.ok)
                    x[v].stg(static_cast<uint8_t *>(p.dx) + r * p.vecs * int64_t(8 * sizeof(T)), at);
            }
        }
        mean = next_mean;
        rstd = next_rstd;
        turn ^= 1;
        if (++slot == g.slots) {
            slot = 0;
            phase ^= 1u;
        }
    }
    row_ring_end(p.status, &flag);
    if (!p.dgamma && !p.dbeta)
        return;
    // The rings are done with: group 0 adds the other groups' sums, in order. [group - 1][2][hidden]
    float *sums = reinterpret_cast<float *>(norm_smem);
    const int hidden = 8 * p.vecs;
    if (g.group > 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (at < p.vecs)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sums[(g.group - 1) * 2 * hidden + 8 * at + i] = dgamma[v][i];
                    sums[((g.group - 1) * 2 + 1) * hidden + 8 * at + i] = dbeta[v][i];
                }
        }
    }
    __syncthreads();
    if (g.group > 0)
        return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int at = g.tid + v * g.threads;
        if (at >= p.vecs)
            continue;
        for (int o = 0; o < p.groups - 1; ++o)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dgamma[v][i] += sums[o * 2 * hidden + 8 * at + i];
                dbeta[v][i] += sums[(o * 2 + 1) * hidden + 8 * at + i];
            }
        float4 *to = reinterpret_cast<float4 *>(p.parts + int64_t(blockIdx.x) * 2 * hidden + 8 * at);
        to[0] = make_float4(dgamma[v][0], dgamma[v][1], dgamma[v][2], dgamma[v][3]);
        to[1] = make_float4(dgamma[v][4], dgamma[v][5], dgamma[v][6], dgamma[v][7]);
        to += hidden / 4;
        to[0] = make_float4(dbeta[v][0], dbeta[v][1], dbeta[v][2], dbeta[v][3]);
        to[1] = make_float4(dbeta[v][4], dbeta[v][5], dbeta[v][6], dbeta[v][7]);
    }
}

// Adds the blocks' sums in a fixed order: a block 32 columns, each warp every eighth part.
constexpr int kNormSumWarps = 8;
__global__ void __launch_bounds__(kNormSumWarps * 32) norm_grad_sum(const __grid_constant__ NormGradParams p) {
    __shared__ float part[kNormSumWarps][32];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hidden = 8 * p.vecs;
    const int col = int(blockIdx.x) * 32 + lane;  // of [2, hidden]
    float sum = 0.0f;
    if (col < 2 * hidden)
#pragma unroll 4
        for (int b = warp; b < p.blocks; b += kNormSumWarps)
            sum += __ldcg(p.parts + int64_t(b) * 2 * hidden + col);
    part[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || col >= 2 * hidden)
        return;
#pragma unroll
    for (int w = 1; w < kNormSumWarps; ++w)
        sum += part[w][lane];
    float *to = col < hidden ? p.dgamma : p.dbeta;
    if (to)
        to[col < hidden ? col : col - hidden] = sum;
}

}  // namespace moe
}  // namespace gg
