// Layer norm of each token and its gradients, and the rounding of rows to 8-bit integers.
//   s = x + residual (rounded to the type)   m = mean s   r = 1 / sqrt(mean (s - m)^2 + eps)   y = (s - m) r gamma + beta
//   ds = r (d - mean d - c mean(d c)) + dsum   with c = (s - m) r, d = dy gamma;   dgamma = sum_t dy c, dbeta = sum_t dy
//
// What bounds them: each row is read once and written once. One block an SM stays for the whole launch; its warps form
// groups that take a row each, one to four vectors of 8 values a thread. Rows come through a ring in shared memory, bulk copies a few rows
// ahead, so that the sums' latency (shuffles and a barrier a row) passes while the next rows are on their way, and a thread's weight, bias
// and sums of gradients stay in registers from row to row. Measured, bf16, with a residual (or its gradient): 16384 x 7168 norm_rows 145-151 us
// (6.2-6.5 TB/s, 95-99% of the measured copy rate), the gradients 161-175 (5.4-5.8 TB/s); 16384 x 4096 85 and 88; fp32 8192 x 4096 90 (forward),
// 2048 x 4096 28 (gradients, of which norm_grad_rows 24).
#pragma once

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kNormMaxHidden = 16384;
constexpr int kNormThreads = 512;      // of a block at most
constexpr int kNormFullThreads = 768;  // of norm_rows' check-free form, which fits 80 registers (fp32 spills 8 bytes; the others 80 to 180)
constexpr int kNormSmem = 212 * 1024;  // of a block's ring and copies at most
constexpr int kNormMaxSlots = 8;       // rows that a group's ring holds
constexpr int kNormMaxGroups = 14;     // each has a named barrier beside the block's own
constexpr int kNormMaxWarps = 16;      // of a group

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
    int params_at;              // the parameters' copy in shared memory, 0: none
    int test_stall;             // test only: 1 = the first slot's barrier waits for an arrival that never comes
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
    int warps, groups, slots, params_at;
    int blocks;
    int test_stall;
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

// Two fp32 values in a 64-bit register pair, and the operations that take both at once (each rounded as the single one).
using pair_t = uint64_t;
__device__ __forceinline__ pair_t pair(float a, float b) {
    pair_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 split(pair_t p) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
    pair_t p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
    pair_t p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
    pair_t p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
    return p;
}
__device__ __forceinline__ float both(pair_t p) {
    const float2 v = split(p);
    return v.x + v.y;
}

// Sums of the two 16-bit values of a word.
template <class T> __device__ __forceinline__ uint32_t plus2(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t plus2<__nv_bfloat16>(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t plus2<__half>(uint32_t a, uint32_t b) {
    const __half2 v = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Eight values of a row in the words that hold them: of 16 bits columns 8 vec to 8 vec + 7, of 32 bits four in the row's first half and
// four in its second (4 vec on, 4 (vecs + vec) on), so that a warp's accesses are 16 bytes a lane side by side.
template <class T> struct Vec8 {
    uint4 w;
    __device__ __forceinline__ void lds(uint32_t row, int vec, int) { w = lds_row(row + uint32_t(vec) * 16u); }
    __device__ __forceinline__ void load(const void *row, int vec, int) { w = static_cast<const uint4 *>(row)[vec]; }
    __device__ __forceinline__ void get(pair_t (&f)[4]) const {
        const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y), c = unpack2<T>(w.z), d = unpack2<T>(w.w);
        f[0] = pair(a.x, a.y), f[1] = pair(b.x, b.y), f[2] = pair(c.x, c.y), f[3] = pair(d.x, d.y);
    }
    __device__ __forceinline__ void set(const pair_t (&f)[4]) {
        const float2 a = split(f[0]), b = split(f[1]), c = split(f[2]), d = split(f[3]);
        w = make_uint4(moe::pack2<T>(a.x, a.y), moe::pack2<T>(b.x, b.y), moe::pack2<T>(c.x, c.y), moe::pack2<T>(d.x, d.y));
    }
    __device__ __forceinline__ void stg(void *row, int vec, int) const { __stcs(static_cast<uint4 *>(row) + vec, w); }
    // Rounded once, and alike, whether the sums are formed in 16 or in 32 bits: where 32 bits do not hold a sum exactly, the smaller term is
    // below a quarter of the larger one's last place.
    __device__ __forceinline__ void add(const Vec8 &o) {
        w = make_uint4(plus2<T>(w.x, o.w.x), plus2<T>(w.y, o.w.y), plus2<T>(w.z, o.w.z), plus2<T>(w.w, o.w.w));
    }
    static __device__ __forceinline__ void stg_q(int8_t *row, int vec, int, uint2 q) { reinterpret_cast<uint2 *>(row)[vec] = q; }
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
    __device__ __forceinline__ void lds(uint32_t row, int vec, int vecs) {
        const uint4 u = lds_row(row + uint32_t(vec) * 16u), v = lds_row(row + uint32_t(vecs + vec) * 16u);
        a = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        b = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ __forceinline__ void load(const void *row, int vec, int vecs) {
        a = static_cast<const float4 *>(row)[vec];
        b = static_cast<const float4 *>(row)[vecs + vec];
    }
    __device__ __forceinline__ void get(pair_t (&f)[4]) const {
        f[0] = pair(a.x, a.y), f[1] = pair(a.z, a.w), f[2] = pair(b.x, b.y), f[3] = pair(b.z, b.w);
    }
    __device__ __forceinline__ void set(const pair_t (&f)[4]) {
        const float2 u = split(f[0]), v = split(f[1]), x = split(f[2]), y = split(f[3]);
        a = make_float4(u.x, u.y, v.x, v.y);
        b = make_float4(x.x, x.y, y.x, y.y);
    }
    __device__ __forceinline__ void stg(void *row, int vec, int vecs) const {
        __stcs(static_cast<float4 *>(row) + vec, a);
        __stcs(static_cast<float4 *>(row) + vecs + vec, b);
    }
    static __device__ __forceinline__ void stg_q(int8_t *row, int vec, int vecs, uint2 q) {
        reinterpret_cast<uint32_t *>(row)[vec] = q.x;
        reinterpret_cast<uint32_t *>(row)[vecs + vec] = q.y;
    }
    __device__ __forceinline__ void add(const Vec8 &o) {
        a = make_float4(a.x + o.a.x, a.y + o.a.y, a.z + o.a.z, a.w + o.a.w);
        b = make_float4(b.x + o.b.x, b.y + o.b.y, b.z + o.b.z, b.w + o.b.w);
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
// the exact quotient, so that the result does not depend on how it is computed. The sum with 1.5 * 2^23 brings a number's nearest whole one
// into the low byte.
//   16-bit values: one in 280 of normal bf16 values is a half exactly, so halves have to come out right on the way. 127 / top = high + low,
//   high cut to so many bits that its products with v and top are exact. m = the whole number near v high; d = v high - m, exact;
//   d' = d + v low, which is the distance from m to within 2^-25 (low's error counts 2e-9 of that) and exactly +-0.5 at a half, while all else is
//   at least 9e-7 away from one (254 v - (2 m + 1) top is a multiple of the last places' product); and m + d' rounds to the even one.
//   32-bit values: v (127 / top) is off by at most 127 * 2 * 2^-24 = 1.5e-5; where that leaves the choice open for one of eight values
//   (within 3e-5 of a half), all eight are decided exactly, by the sign of 254 v - (2 f + 1) top, f = floor: both products are split into a rounded
//   part and its error by fma, and their difference is exact (it is small).
// Rows whose top is below 2^-60 or above 2^60 are decided that way, too, scaled by 2^80 or 2^-80 first so that nothing leaves fp32's normal range.
// A row of zeros has scale 0 and q 0; one that holds NaN or an infinity has scale NaN and q 0.
// (32768 bf16 rows of 7168: each value by itself, with a conversion and the test for a half, 230 us; decided as fp32 is 160; this 116.)
template <class T> struct Rounding {
    static constexpr bool kShort = sizeof(T) == 2;
    static constexpr uint32_t kHigh = std::is_same<T, __half>::value ? 0xfffff800u : 0xffffff00u;  // 13 + 11 or 16 + 8 bits of a product
    float top, inverse, low, up;
    bool zero, careful;  // all q are 0; all values the exact way
    static __device__ __forceinline__ float scale(uint32_t top_bits) {
        return top_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(top_bits), 127.0f);
    }
    __device__ __forceinline__ explicit Rounding(uint32_t top_bits) {  // of the largest magnitude's bits (NaN above all)
        top = __uint_as_float(top_bits);
        zero = top_bits >= 0x7f800000u || top_bits == 0u;
        up = top < 8.6736174e-19f ? 1.2089258e24f : top > 1.1529215e18f ? 8.2718061e-25f : 1.0f;  // 2^-60, 2^80; 2^60, 2^-80
        careful = zero || up != 1.0f;
        top = zero ? 1.0f : top * up;
        const float r = __frcp_rn(top);
        inverse = 127.0f * r;
        if constexpr (kShort) {
            const float high = __uint_as_float(__float_as_uint(inverse) & kHigh);
            low = fmaf(-high, top, 127.0f) * r;
            if (!careful)
                inverse = high;
        }
    }
    __device__ __forceinline__ uint32_t exact(float v) const {
        if (zero)
            return 0u;
        const float a = fabsf(v) * up, t = a * inverse;
        float m = rintf(t);
        if (fabsf(t - m) > 0.49997f) {
            const float f = floorf(t), b = 2.0f * f + 1.0f, p = b * top;
            const float e = fmaf(b, top, -p), r = fmaf(254.0f, a, -p);
            m = r > e ? f + 1.0f : r < e ? f : 2.0f * rintf(0.5f * (f + 0.5f));
        }
        return uint32_t(v < 0.0f ? -int(m) : int(m));
    }
    __device__ __forceinline__ uint2 operator()(const pair_t (&v)[4]) const {
        uint32_t n[8];
        float worst = 0.0f;
        const pair_t by = pair(inverse, inverse), to_low = pair(12582912.0f, 12582912.0f), minus = pair(-1.0f, -1.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pair_t s = fma2(v[i], by, to_low);
            pair_t off = fma2(v[i], by, fma2(s, minus, to_low));
            if constexpr (kShort) {
                off = fma2(v[i], pair(low, low), off);
                s = add2(s, off);
            } else {
                const float2 o = split(off);
                worst = fmaxf(worst, fmaxf(fabsf(o.x), fabsf(o.y)));
            }
            const float2 bits = split(s);
            n[2 * i] = __float_as_uint(bits.x);
            n[2 * i + 1] = __float_as_uint(bits.y);
        }
        if (careful || (!kShort && worst > 0.49997f))
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = split(v[i]);
                n[2 * i] = exact(f.x);
                n[2 * i + 1] = exact(f.y);
            }
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
// longer is read again. part: 16 words of shared memory, other ones for the next row. before() runs before the block's one barrier, then
// to(scale) says where rows go: what it returns takes (vec, vecs, eight integers).
constexpr int kQuantHeld = 4;
template <class T, class B, class S> __device__ __forceinline__ void quant_row(const void *row, int vecs, uint32_t *part, B &&before, S &&to) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    Vec8<T> v[kQuantHeld];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i) {
        const int at = tid + i * int(blockDim.x);
        if (at < vecs)
            v[i].load(row, at, vecs);
    }
    before();
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i)
        if (tid + i * int(blockDim.x) < vecs)
            top = v[i].top(top);
    for (int at = tid + kQuantHeld * int(blockDim.x); at < vecs; at += blockDim.x) {
        Vec8<T> u;
        u.load(row, at, vecs);
        top = u.top(top);
    }
    top = __reduce_max_sync(0xffffffffu, Vec8<T>::bits(top));
    if (lane == 0)
        part[warp] = top;
    __syncthreads();  // a warp writes these words again only after the next row's barrier
    top = __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
    const Rounding<T> by(top);
    auto store = to(tid == 0 ? Rounding<T>::scale(top) : 0.0f);
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i) {
        const int at = tid + i * int(blockDim.x);
        if (at < vecs) {
            pair_t f[4];
            v[i].get(f);
            store(at, vecs, by(f));
        }
    }
    for (int at = tid + kQuantHeld * int(blockDim.x); at < vecs; at += blockDim.x) {
        Vec8<T> u;
        pair_t f[4];
        u.load(row, at, vecs);
        u.get(f);
        store(at, vecs, by(f));
    }
}
// To one place.
template <class T> __device__ __forceinline__ void quant_row(const void *row, int8_t *q, float *scale_to, int vecs, uint32_t *part) {
    quant_row<T>(row, vecs, part, [] {}, [&](float scale) {
        if (threadIdx.x == 0)
            *scale_to = scale;
        return [=](int at, int n, uint2 v) { Vec8<T>::stg_q(q, at, n, v); };
    });
}

// A block a row (and every gridDim.x-th after it). 32768 rows of 7168, bf16: 116-124 us (5.7-6.1 TB/s).
template <class T> __global__ void __launch_bounds__(512) quant_rows(const __grid_constant__ QuantParams p) {
    __shared__ uint32_t part[2][16];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    int turn = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1)
        quant_row<T>(static_cast<const uint8_t *>(p.x) + r * p.vecs * int64_t(8 * sizeof(T)), p.q + r * p.vecs * 8, p.scales + r, p.vecs, part[turn]);
}

// ---- sums of two values at a time ----

// Of a warp: lanes 0-15 get the sum of a, lanes 16-31 that of b.
__device__ __forceinline__ float halves_sum(float a, float b) {
    const bool low = (threadIdx.x & 16u) == 0;
    float keep = low ? a : b;
    keep += __shfl_xor_sync(0xffffffffu, low ? b : a, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
        keep += __shfl_xor_sync(0xffffffffu, keep, o);
    return keep;
}
// Of each half warp's 16 values, both sums for all lanes.
__device__ __forceinline__ float2 each_half_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
}

// ---- rows through a ring in shared memory ----

// A group of warps of a block, its ring of rows and its barrier. All threads of a group take the same steps; a wait that gives up is
// recorded and the group goes on without waiting, so that its barriers stay matched.
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
            ptx::mbar_init(g.bars + 8u * s, p.test_stall && blockIdx.x == 0 && g.group == 0 && s == 0 ? 2 : 1);
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

// A thread's weights or biases, 8 a vector: held in registers for all rows where it has one or two vectors, else read for each row from
// the block's copy in shared memory (or, where there is no place for that, from global memory), since they would cost the registers
// that hold the row or the sums.
template <class T, class W, int V> struct NormParam {
    static constexpr bool kHeld = V <= 2;
    const uint8_t *from;  // null: 1 or 0 throughout
    float otherwise;
    int vecs;
    Vec8<W> held[kHeld ? V : 1];
    // copy: place in shared memory, or null. By all threads of the block, which have to be together before the first use.
    __device__ __forceinline__ NormParam(const void *array, float otherwise_, int first, int step, int vecs_, uint8_t *copy)
        : from(static_cast<const uint8_t *>(array)), otherwise(otherwise_), vecs(vecs_) {
        if constexpr (kHeld) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (first + v * step < vecs)
                    read(held[v], first + v * step);
        } else if (array && copy) {
            for (int i = threadIdx.x; i < vecs * int(sizeof(W)) / 2; i += blockDim.x)
                reinterpret_cast<uint4 *>(copy)[i] = __ldcg(static_cast<const uint4 *>(array) + i);
            from = copy;
        }
    }
    __device__ __forceinline__ void read(Vec8<W> &v, int at) const {
        if (!from) {
            const pair_t both = pair(otherwise, otherwise), all[4] = {both, both, both, both};
            v.set(all);
            return;
        }
        const uint4 *words = reinterpret_cast<const uint4 *>(from);
        if constexpr (std::is_same<W, float>::value) {
            constexpr bool near = !std::is_same<T, float>::value;  // the columns of a 16-bit row's vector
            const uint4 a = words[near ? 2 * at : at], b = words[near ? 2 * at + 1 : vecs + at];
            v.a = make_float4(__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w));
            v.b = make_float4(__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w));
        } else {
            v.w = words[at];
        }
    }
    __device__ __forceinline__ void get(int v, int at, pair_t (&f)[4]) const {
        if constexpr (kHeld) {
            held[v].get(f);
        } else {
            Vec8<W> w;
            read(w, at);
            w.get(f);
        }
    }
};

// What a row's values are moved by: where their squares pass fp32 (rstd 0) their distance to the mean can pass it, too, and 0 times that would not be 0.
__device__ __forceinline__ float minus_mean_of(float mean, float rstd) { return rstd == 0.0f && fabsf(mean) < INFINITY ? 0.0f : -mean; }

// kFull: every thread has V vectors, so that none asks for each (only with four: with two it saved the forward pass instructions but took
// 157 us in place of 145 for 16384 x 7168 with a residual, its reads and writes closer together).
// Forward it takes more groups of warps at once (kNormFullThreads): with 8-bit rows, whose way is long and has two barriers, 16384 rows of 7168
// take 123-125 us with three groups of seven warps (136 with two), of 12288 191 with two of twelve (240 with one), of 4096 68 (71). Where the groups
// stay as many, the fewer registers cost up to 4% (16384 columns 290 against 280). Four groups in 72 registers won nothing at 7168 and lost 5% at
// 5120 and 8192.
// Mean and variance without cancellation: each warp its own mean m_w and the squares S_w around it, joined around the first warp's mean, t_w = m_w - m_0:
//   mean = m_0 + sum n_w t_w / n     sum (v - mean)^2 = sum (S_w + n_w t_w^2) - n (mean - m_0)^2
// where what is taken off is at most the sum of the others' n_w t_w^2, so that no more than a factor of the number of warps is lost.
// Where one of these sums passes fp32, the row is joined once more by the warps' shares n_w / n, which pass it only where the row's own squares do:
// means of 8 values or more are far from fp32's end, and where a t_w^2 passes it, the squares around the row's mean, 4 t_w^2 at least, do too.
template <class T, class W, int V, bool kFull>
__global__ void __launch_bounds__(kFull ? kNormFullThreads : kNormThreads, 1) norm_rows(const __grid_constant__ NormParams p) {
    extern __shared__ __align__(1024) uint8_t norm_smem[];
    __shared__ uint64_t bars[kNormMaxGroups * kNormMaxSlots];
    __shared__ float part[kNormMaxGroups][2][2 * kNormMaxWarps];
    __shared__ uint32_t tops[kNormMaxGroups][2][kNormMaxWarps];
    __shared__ volatile uint32_t flag;
    RowRing<2> g = row_ring<2>(p, p.residual ? 2 : 1, ptx::smem_addr(norm_smem), bars, &flag, p.vecs * int(8 * sizeof(T)));
    g.from[0] = static_cast<const uint8_t *>(p.x);
    g.from[1] = static_cast<const uint8_t *>(p.residual);
    const int warp = g.tid >> 5, lane = g.tid & 31;
    for (int s = 0; s < g.slots; ++s)
        g.load(s, g.first + s * g.stride);
    // values of warp w
    auto count = [&](int w) {
        int n = 0;
#pragma unroll
        for (int v = 0; v < V; ++v)
            n += min(32, max(0, p.vecs - v * g.threads - w * 32));
        return float(8 * n);
    };
    const float inv_mine = 1.0f / fmaxf(8.0f, count(warp)), hidden = float(8 * p.vecs), inv_hidden = 1.0f / hidden;
    const int other = lane & 15;  // the warp whose sums this lane joins
    const float theirs = other < p.warps ? count(other) : 0.0f;
    const int param_bytes = p.vecs * int(8 * sizeof(W));
    uint8_t *copy = p.params_at ? norm_smem + p.params_at : nullptr;
    const NormParam<T, W, V> gamma(p.gamma, 1.0f, g.tid, g.threads, p.vecs, copy),
        beta(p.beta, 0.0f, g.tid, g.threads, p.vecs, copy ? copy + param_bytes : nullptr);
    __syncthreads();
    int slot = 0, turn = 0;
    uint32_t phase = 0;
    for (int64_t r = g.first; r < p.rows; r += g.stride) {
        g.wait(slot, phase);
        const int64_t row = r * g.row_bytes;
        pair_t f[V][4];
        pair_t sum = 0;  // of even and of odd columns
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (kFull || at < p.vecs) {
                Vec8<T> x;
                x.lds(g.at(slot, 0), at, p.vecs);
                if (p.residual) {
                    Vec8<T> more;
                    more.lds(g.at(slot, 1), at, p.vecs);
                    x.add(more);
                    if (p.sum)
                        x.stg(static_cast<uint8_t *>(p.sum) + row, at, p.vecs);
                }
                x.get(f[v]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum = add2(sum, f[v][i]);
            }
        }
        const float m_warp = warp_sum(both(sum)) * inv_mine;
        const pair_t minus_warp = pair(-m_warp, -m_warp);
        pair_t squared = 0;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (kFull || g.tid + v * g.threads < p.vecs)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const pair_t d = add2(f[v][i], minus_warp);
                    squared = fma2(d, d, squared);
                }
        const float squares = warp_sum(both(squared));
        float *box = part[g.group][turn];
        if (lane == 0) {
            box[warp] = m_warp;
            box[kNormMaxWarps + warp] = squares;
        }
        g.sync();  // the slot has been read, too
        g.load(slot, r + g.slots * g.stride);
        const float m_first = box[0];
        const float t = other < p.warps ? box[other] - m_first : 0.0f;
        const float2 joined = each_half_sum(lane < 16 ? theirs * t : other < p.warps ? fmaf(theirs * t, t, box[kNormMaxWarps + other]) : 0.0f);
        const float off = joined.x * inv_hidden;
        float mean = m_first + off, minus = -mean, rstd = rsqrtf(fmaxf(0.0f, joined.y * inv_hidden - off * off) + p.eps);
        if (!(joined.y < INFINITY)) {  // (joined.x passes fp32 only where joined.y does) alike in all of a group's threads
            const float share = theirs * inv_hidden, of_warp = other < p.warps ? box[kNormMaxWarps + other] : 0.0f;
            const float2 far = each_half_sum(lane < 16 ? share * t : fmaf(share * t, t, of_warp * inv_hidden));
            mean = box[0] + far.x;
            const float var = fmaxf(0.0f, far.y - far.x * far.x), squares = far.y < INFINITY ? var * hidden : far.y;
            rstd = rsqrtf(squares < INFINITY ? var + p.eps : squares);  // infinite squares: 0, and NaN stays
            minus = minus_mean_of(mean, rstd);
        }
        if (g.tid == 0 && g.ok) {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
        uint32_t top = 0;
        Vec8<T> y[V];
        // (s rstd - mean rstd would be one operation less, but off by a rounding of mean rstd: rows of one value would not give beta)
        const pair_t minus_mean = pair(minus, minus), both_rstd = pair(rstd, rstd);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (kFull || at < p.vecs) {
                pair_t a[4], b[4];
                gamma.get(v, at, a);
                beta.get(v, at, b);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    f[v][i] = fma2(mul2(add2(f[v][i], minus_mean), both_rstd), a[i], b[i]);
                y[v].set(f[v]);
                if (p.y)
                    y[v].stg(static_cast<uint8_t *>(p.y) + row, at, p.vecs);
                if (p.q)
                    top = y[v].top(top);
            }
        }
        if (p.q) {
            uint32_t *most = tops[g.group][turn];
            top = __reduce_max_sync(0xffffffffu, Vec8<T>::bits(top));
            if (lane == 0)
                most[warp] = top;
            g.sync();
            top = __reduce_max_sync(0xffffffffu, lane < p.warps ? most[lane] : 0u);
            const Rounding<T> by(top);
            if (g.tid == 0 && g.ok)
                p.q_scales[r] = Rounding<T>::scale(top);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int at = g.tid + v * g.threads;
                if (kFull || at < p.vecs) {
                    pair_t a[4];
                    y[v].get(a);  // the integers are of y as it is written
                    Vec8<T>::stg_q(p.q + r * p.vecs * 8, at, p.vecs, by(a));
                }
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
// leaves its sums for norm_grad_sum. A row is read from its slot twice, before and after the sums along it, so that the registers hold
// those sums only; so a slot is loaded again one row later, when the next row's barrier shows that all are past it.
template <class T, class W, int V, bool kFull>
__global__ void __launch_bounds__(kNormThreads, 1) norm_grad_rows(const __grid_constant__ NormGradParams p) {
    extern __shared__ __align__(1024) uint8_t norm_smem[];
    __shared__ uint64_t bars[kNormMaxGroups * kNormMaxSlots];
    __shared__ float part[kNormMaxGroups][2][2 * kNormMaxWarps];
    __shared__ volatile uint32_t flag;
    RowRing<3> g = row_ring<3>(p, p.dsum ? 3 : 2, ptx::smem_addr(norm_smem), bars, &flag, p.vecs * int(8 * sizeof(T)));
    g.from[0] = static_cast<const uint8_t *>(p.x);
    g.from[1] = static_cast<const uint8_t *>(p.dy);
    g.from[2] = static_cast<const uint8_t *>(p.dsum);
    const int warp = g.tid >> 5, lane = g.tid & 31;
    for (int s = 0; s < g.slots; ++s)
        g.load(s, g.first + s * g.stride);
    const float inv_hidden = 1.0f / float(8 * p.vecs);
    const NormParam<T, W, V> gamma(p.gamma, 1.0f, g.tid, g.threads, p.vecs, p.params_at ? norm_smem + p.params_at : nullptr);
    __syncthreads();
    pair_t dgamma[V][4] = {}, dbeta[V][4] = {};
    float next_mean = 0.0f, next_rstd = 0.0f;
    if (g.first < p.rows) {
        next_mean = __ldcg(p.mean + g.first);
        next_rstd = __ldcg(p.rstd + g.first);
    }
    int slot = 0, turn = 0;
    uint32_t phase = 0;
    for (int64_t r = g.first; r < p.rows; r += g.stride) {
        const float rstd = next_rstd;
        const float minus = minus_mean_of(next_mean, rstd);
        const pair_t minus_mean = pair(minus, minus), both_rstd = pair(rstd, rstd);
        if (r + g.stride < p.rows) {
            next_mean = __ldcg(p.mean + r + g.stride);
            next_rstd = __ldcg(p.rstd + r + g.stride);
        }
        g.wait(slot, phase);
        pair_t along = 0, level = 0;  // sums of d c and of d, of even and of odd columns
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (kFull || at < p.vecs) {
                Vec8<T> x, dy;
                pair_t a[4], b[4], w[4];
                x.lds(g.at(slot, 0), at, p.vecs);
                dy.lds(g.at(slot, 1), at, p.vecs);
                x.get(a);
                dy.get(b);
                gamma.get(v, at, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const pair_t c = mul2(add2(a[i], minus_mean), both_rstd), d = mul2(b[i], w[i]);
                    level = add2(level, d);
                    along = fma2(d, c, along);
                    dgamma[v][i] = fma2(b[i], c, dgamma[v][i]);
                    dbeta[v][i] = add2(dbeta[v][i], b[i]);
                }
            }
        }
        const float mine = halves_sum(both(along), both(level));
        float *box = part[g.group][turn];
        if ((lane & 15) == 0)
            box[(lane & 16) + warp] = mine;  // kNormMaxWarps of each
        g.sync();  // all are past the row before
        if (g.slots > 1 && r != g.first)
            g.load(slot ? slot - 1 : g.slots - 1, r + (g.slots - 1) * g.stride);
        const float2 sums = each_half_sum((lane & 15) < p.warps ? box[lane] : 0.0f);
        // dx = rstd (d + (x - mean) tilt) + less: no factor of it is the square of rstd or of a value
        const float less = -rstd * (sums.y * inv_hidden), tilt = -rstd * (sums.x * inv_hidden);
        const pair_t both_less = pair(less, less), slope = pair(tilt, tilt);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (kFull || at < p.vecs) {
                Vec8<T> x, dy;
                pair_t a[4], b[4], w[4];
                x.lds(g.at(slot, 0), at, p.vecs);
                dy.lds(g.at(slot, 1), at, p.vecs);
                x.get(a);
                dy.get(b);
                gamma.get(v, at, w);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a[i] = fma2(fma2(add2(a[i], minus_mean), slope, mul2(b[i], w[i])), both_rstd, both_less);
                if (p.dsum) {
                    x.lds(g.at(slot, 2), at, p.vecs);
                    x.get(b);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        a[i] = add2(a[i], b[i]);
                }
                x.set(a);
                x.stg(static_cast<uint8_t *>(p.dx) + r * g.row_bytes, at, p.vecs);
            }
        }
        if (g.slots == 1) {
            g.sync();
            g.load(0, r + g.stride);
        }
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
    auto of_group = [&](int o, int which, int vec) { return reinterpret_cast<ulonglong2 *>(sums + (2 * o + which) * hidden + 8 * vec); };
    if (g.group > 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = g.tid + v * g.threads;
            if (kFull || at < p.vecs)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    of_group(g.group - 1, 0, at)[i] = make_ulonglong2(dgamma[v][2 * i], dgamma[v][2 * i + 1]);
                    of_group(g.group - 1, 1, at)[i] = make_ulonglong2(dbeta[v][2 * i], dbeta[v][2 * i + 1]);
                }
        }
    }
    __syncthreads();
    if (g.group > 0)
        return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int at = g.tid + v * g.threads;
        if (!kFull && at >= p.vecs)
            continue;
        for (int o = 0; o < p.groups - 1; ++o)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const ulonglong2 a = of_group(o, 0, at)[i], b = of_group(o, 1, at)[i];
                dgamma[v][2 * i] = add2(dgamma[v][2 * i], a.x);
                dgamma[v][2 * i + 1] = add2(dgamma[v][2 * i + 1], a.y);
                dbeta[v][2 * i] = add2(dbeta[v][2 * i], b.x);
                dbeta[v][2 * i + 1] = add2(dbeta[v][2 * i + 1], b.y);
            }
        ulonglong2 *to = reinterpret_cast<ulonglong2 *>(p.parts + int64_t(blockIdx.x) * 2 * hidden);
        constexpr bool split_row = std::is_same<T, float>::value;  // see Vec8
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int four = split_row ? at + i * p.vecs : 2 * at + i;
            to[four] = make_ulonglong2(dgamma[v][2 * i], dgamma[v][2 * i + 1]);
            to[hidden / 4 + four] = make_ulonglong2(dbeta[v][2 * i], dbeta[v][2 * i + 1]);
        }
    }
}

// Adds the blocks' sums in a fixed order: a block 32 columns, each warp every eighth part. (With 10 or 19 parts on
// their way at once it takes 0.8 to 1.7 us longer: its registers no longer fit beside the blocks whose end it waits for.)
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
