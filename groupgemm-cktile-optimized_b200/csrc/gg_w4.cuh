// Rows in expert order times their expert's 4-bit weights with group scales, for few rows an expert:
//   out[r, n] = sum over groups g of scale[e, n, g] * sum_{k in g} (q[e, n, k] - zero[e, n, g]) x[row(r), k]
//
// What bounds it: the weights are read once, 1/2 byte each, and at HBM's rate that is 46 weights a
// cycle and SM: the arithmetic that makes a 16-bit operand of each is what has to keep up. So each
// weight is widened once, by the thread that owns its row, whatever the number of tokens, and
// the products go to the tensor cores from Tensor Memory:
//
//   warp 0       TMA: 256 weight rows x 128 k (16 KB, 64-byte swizzle) a step into a shared-memory ring
//   warp 3       a bulk copy of the tokens' 128 k a step (w4_gather lays them out so beforehand, see there)
//   warps 4-11   a group of four for each half of the weight rows, a thread a row: 16 bytes at a time from the ring,
//                widened to q - zero (exact) in registers, tcgen05.st into the half's next A operand
//   warps 1, 2   a half each: tcgen05.mma, D[weight row, token] = A (Tensor Memory) x B (tokens), a fresh accumulator
//                a group
//   warps 12-19  a half each four: tcgen05.ld of a step's products and the fp32 sum with the group's scale (one scalar a
//                thread); output
//
// Three A operands and two D a half keep the widening from waiting for the MMAs: beside four widening warps a scheduler the
// MMA warp's eight take 530 cycles to issue, against 95 alone. (Also built: mma.sync m16n8k16 from registers, 54 / 139 / 693 us on
// one token, 148 and 1024 rows: above 8 tokens it is bound by its own rate, 11 cycles a scheduler; and four
// groups that widen odd and even steps with an A operand each and add up themselves, 45 / 104 / 361 us.)
//
// Work split: the steps of all (expert, token chunk, 256-row tile) items in a row, dealt out to the CTAs in
// equal contiguous ranges, so that one token through a few experts still keeps every SM reading. A tile that is
// cut leaves fp32 partial sums in the workspace; the CTA that arrives last adds them in order of k.
#pragma once

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kW4Threads = 640;
constexpr int kW4TileRows = 256;
constexpr int kW4StepK = 128;
constexpr int kW4MaxExperts = 1024;
constexpr int kW4WeightBytes = kW4TileRows * kW4StepK / 2;

struct W4Params {
    const void *x;           // [tokens or rows, k]
    const void *scales;      // [experts, n, groups]
    const uint8_t *zeros;    // [experts, n, groups] or null = 8
    const int32_t *offsets;  // [experts + 1]
    const int32_t *src;      // [rows] slots, or null: row r reads x[r]
    void *out;               // [rows, n]
    uint32_t *status;        // [0] status word, [2] timeouts of this launch
    uint8_t *xs;             // [rows + 8 experts][steps] 256 bytes: the rows of x as the products read them
    float *ws;               // [2 x grid][tokens of a chunk][256] partial sums
    int32_t *counters;       // [grid] arrivals at a cut tile, 0 between launches
    int64_t rows, slots;     // slots: tokens * top_k
    uint64_t timeout_ns;
    int n, k, groups, experts, top_k, tiles, steps;  // steps: of 128 k
    int chunk;       // tokens of a chunk
};

// Tokens of a chunk: at most 32 (a thread holds a sum a token). Tensor Memory's 512 columns hold for each half kA operands of
// 64 columns and two D of a column a token and group of a step.
template <int G> struct W4Cfg {
    static constexpr int kSub = kW4StepK / G;  // groups a step
    static constexpr int kTokens = kSub == 4 ? 16 : 32;
    static constexpr int kA = kSub == 1 ? 3 : 2;
    static constexpr int kD = kSub * kTokens;  // columns of a D
    static constexpr int kStageBytes = kW4WeightBytes + kTokens * kW4StepK * 2;
    static constexpr int kStages = 6;  // a multiple of 2 and of kA: a stage always meets the same D and A
    static constexpr int kBars = 4 * kStages + 4 * kA + 4;
    static constexpr int kTableBytes = 2 * (kW4MaxExperts + 1) * 4;
    static_assert(2 * (64 * kA + 2 * kD) <= 512 && kStages % kA == 0 && kStages % 2 == 0, "Tensor Memory");
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kBars * 8 + kTableBytes + 64;
};

// ---- instructions this kernel adds to gg_ptx.cuh's ----

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16],"
                 " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
// One step's eight MMAs of 16 k for 128 weight rows: D (Tensor Memory) = A (Tensor Memory, two 16-bit values a column)
// x B (shared memory, descriptor hi:lo), a D of its own for each group of G. Issued where pred != 0. In one block with
// addresses one add away from its operands, in a loop that is not unrolled: with the stages unrolled and every address a constant the
// warps of the other roles stalled three issue slots of four on the instruction cache.
#define GG_W4_MMA(i, acc) \
    "add.u32 d, %0, " #i "*16/%8*%7;\n\tadd.u32 a, %1, " #i "*8;\n\tadd.u32 l, %2, " #i "/4*%6+(" #i "&3)*2;\n\tmov.b64 b, {l, %3};\n\t" \
    "@q tcgen05.mma.cta_group::1.kind::f16 [d], [a], b, %4, " acc ";\n\t"
template <int G, int kTokens>
__device__ __forceinline__ void w4_mma_step(uint32_t d, uint32_t a, uint32_t lo, uint32_t hi, uint32_t idesc, uint32_t pred) {
#define GG_W4_STEP(a1, a2, a3, a4, a5, a6, a7)                                                                                          \
    asm volatile("{\n\t.reg .pred q, t, f;\n\t.reg .b32 d, a, l;\n\t.reg .b64 b;\n\tsetp.ne.b32 q, %5, 0;\n\t"                            \
                 "setp.eq.b32 t, 0, 0;\n\tsetp.ne.b32 f, 0, 0;\n\t" GG_W4_MMA(0, "f") GG_W4_MMA(1, a1) GG_W4_MMA(2, a2) GG_W4_MMA(3, a3) \
                     GG_W4_MMA(4, a4) GG_W4_MMA(5, a5) GG_W4_MMA(6, a6) GG_W4_MMA(7, a7) "}" ::"r"(d),                                  \
                 "r"(a), "r"(lo), "r"(hi), "r"(idesc), "r"(pred), "n"(kTokens * 128 / 16), "n"(kTokens), "n"(G)                         \
                 : "memory")
    if constexpr (G == 128)
        GG_W4_STEP("t", "t", "t", "t", "t", "t", "t");
    else if constexpr (G == 64)
        GG_W4_STEP("t", "t", "t", "f", "t", "t", "t");
    else
        GG_W4_STEP("t", "f", "t", "f", "t", "f", "t");
#undef GG_W4_STEP
}
#undef GG_W4_MMA
// `bytes` (a multiple of 16) from global to shared memory, counted on an mbarrier; where pred != 0.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, uint32_t pred) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar), "r"(pred)
                 : "memory");
}
__device__ __forceinline__ void named_sync(int bar, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Four bits as a 16-bit float without a conversion or a power of two to put them on: where a format's exponent field is 0 or
// 1 its value is linear in its bits, i * 2^-24 (fp16, i below 2048) and i * 2^-133 (bf16, i below 256). So a masked nibble in bits
// 0-3 or 4-7 is q or 16 q times that unit, and one fma by a power of two brings both to (q - zero) * W4Unit::kValue, exactly (the
// subnormal inputs are not flushed by it). bf16 cannot reach 1 in one multiplication, so its weights stay in units of 2^-9, which
// the group's scale takes back in fp32. A word costs 5 instructions on the ALU pipe (one shift, four masks) and 4 on the
// FMA pipe; with powers of two or'ed in, bf16 had needed 7 and 4: 150 ns for a warp's step of 32 rows x 128 k against 111.
template <class T> struct W4Unit;
template <> struct W4Unit<__half> {
    static constexpr uint32_t kLow = 0x6c006c00u;     // 2^12: with kHigh 2^8, weights in units of 2^-12
    static constexpr uint32_t kHigh = 0x5c005c00u;    // 2^8
    static constexpr float kBack = 4096.0f;
};
template <> struct W4Unit<__nv_bfloat16> {
    static constexpr uint32_t kLow = 0x7d807d80u;     // 2^124
    static constexpr uint32_t kHigh = 0x7b807b80u;    // 2^120
    static constexpr float kBack = 512.0f;
};
template <class T> __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c);
template <> __device__ __forceinline__ uint32_t fma2<__half>(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
template <> __device__ __forceinline__ uint32_t fma2<__nv_bfloat16>(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// -zero in the weights' unit, twice.
template <class T> __device__ __forceinline__ uint32_t w4_minus(uint32_t zero) {
    return fma2<T>(zero * 0x00010001u, W4Unit<T>::kLow ^ 0x80008000u, 0u);
}
// The eight weights of a word as four pairs (k, k + 4): the pairs that masks and shifts of the whole word give. Each
// eight values of x are put into that order, so the products pair up.
template <class T> __device__ __forceinline__ void widen(uint32_t w, uint32_t minus, uint32_t *out) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t v = w >> (8 * j);
        out[2 * j] = fma2<T>(v & 0x000f000fu, W4Unit<T>::kLow, minus);
        out[2 * j + 1] = fma2<T>(v & 0x00f000f0u, W4Unit<T>::kHigh, minus);
    }
}

// Bounded wait of a converged warp, as wait_all, with a hint that lets the hardware hold the thread: twenty warps wait
// here in turn, and their polling would take issue slots from the widening.
__device__ __forceinline__ bool try_wait_hint(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity), "r"(10000)
                 : "memory");
    return ok != 0;
}
__device__ __noinline__ inline bool w4_wait_slow(uint32_t bar, uint32_t parity, const Abort ab, uint32_t code) {
    const uint64_t t0 = ptx::globaltimer();
    for (uint32_t it = 1;; ++it) {
        if (__all_sync(0xffffffffu, try_wait_hint(bar, parity)))
            return true;
        if ((it & 15u) == 0) {
            bool stop = *ab.flag != 0u || *(volatile uint32_t *)ab.status != 0u;
            if (!stop && ptx::globaltimer() - t0 > ab.timeout_ns) {
                atomicCAS(ab.status, 0u, code);
                stop = true;
            }
            if (__any_sync(0xffffffffu, stop)) {
                *ab.flag = 1u;
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool w4_wait(uint32_t bar, uint32_t parity, const Abort &ab, uint32_t code) {
    return __all_sync(0xffffffffu, try_wait_hint(bar, parity)) || w4_wait_slow(bar, parity, ab, code);
}
// A look at a barrier ahead of the wait for it, so that its latency passes behind other work: `seen` goes to w4_wait_seen.
__device__ __forceinline__ bool look(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool w4_wait_seen(bool seen, uint32_t bar, uint32_t parity, const Abort &ab, uint32_t code) {
    return __all_sync(0xffffffffu, seen) || w4_wait_slow(bar, parity, ab, code);
}

// The launch's work: items in expert order, an item's steps in order of k.
struct W4Item {
    int e, n0, r0, count;
};
__device__ __forceinline__ W4Item w4_item(const W4Params &p, const int *start, const int *first, int64_t item, int chunk_tokens) {
    // the last expert whose first chunk's items start at or before the item
    int lo = 0, hi = p.experts - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (int64_t(first[mid]) * p.tiles <= item)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int chunks = first[lo + 1] - first[lo];
    const int at = int(item - int64_t(first[lo]) * p.tiles);
    const int tile = at / chunks, chunk = at - tile * chunks;
    const int r0 = start[lo] + chunk * chunk_tokens;
    return {lo, tile * kW4TileRows, r0, min(chunk_tokens, start[lo + 1] - r0)};
}
__device__ __forceinline__ int w4_cta_of(int64_t step, int64_t total, int ctas) { return int(((step + 1) * ctas - 1) / total); }

// offsets come from the device: each is held to the range that the rows allow
__device__ __forceinline__ void w4_starts(const W4Params &p, int *start) {
    for (int e = threadIdx.x; e <= p.experts; e += blockDim.x) {
        const int64_t v = p.offsets[e], before = e ? p.offsets[e - 1] : 0;
        if (v < before || v > p.rows || before < 0)
            report(p.status, kSiteOffsets);
        start[e] = int(max(int64_t(0), min(v, p.rows)));
    }
}

// The rows of x in expert order, gathered through src, as the products read them: for each chunk of `chunk` tokens of an
// expert and each step of 128 k a shared-memory image of B (K-major, two halves of 64 k, each a row of 128 bytes a token with the
// 128-byte swizzle; token count rounded up to 8) so that a bulk copy a half loads it; eight values at a time in the order
// in which masks and shifts take the weights out of a word. One 16-byte piece a thread. (Done by warps of the product
// kernel instead, with cp.async and shared memory, this took them 1400 cycles a step at 16 tokens: twice what HBM allows.) Rows of
// no expert are set to zero in out.
constexpr int kW4GatherThreads = 128;
template <class T> __global__ void __launch_bounds__(kW4GatherThreads) w4_gather(const __grid_constant__ W4Params p) {
    __shared__ int start[kW4MaxExperts + 1];
    ptx::griddep_wait();
    // The product kernel may start now. It reads what earlier kernels wrote (offsets, scales, weights) without waiting for this one
    // to end: every block of this one has passed its own wait by then. Before it reads xs it waits for this one.
    ptx::griddep_launch_dependents();
    w4_starts(p, start);
    __syncthreads();
    const int piece = int(blockIdx.y) * kW4GatherThreads + int(threadIdx.x);  // of a row: 8 values
    const int step = piece >> 4, half = (piece >> 3) & 1, c = piece & 7;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        if (r < start[0] || r >= start[p.experts]) {
            for (int col = piece; col < p.n; col += int(gridDim.y) * kW4GatherThreads)
                static_cast<T *>(p.out)[r * p.n + col] = from_f32<T>(0.0f);
            continue;
        }
        if (step >= p.steps)
            continue;
        int lo = 0, hi = p.experts - 1;  // the last expert that starts at or before the row
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (start[mid] <= r)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int in_expert = int(r) - start[lo], i = in_expert % p.chunk;
        const int count = (min(p.chunk, start[lo + 1] - (int(r) - i)) + 7) & ~7;
        if (i >= count)
            continue;  // falling offsets, reported
        int64_t row = r;
        if (p.src) {
            const int s = p.src[r];
            row = s < 0 || s >= p.slots ? -1 : s / p.top_k;
            if (row < 0 && piece == 0)
                report(p.status, kSiteSrc);
        }
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row >= 0 && piece * 8 < p.k)
            v = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.x) + row * p.k + piece * 8);
        const int64_t base = int64_t(int(r) - i + 8 * lo) * p.steps * 256;
        *reinterpret_cast<uint4 *>(p.xs + base + (int64_t(step * 2 + half) * count + i) * 128 + ((c ^ (i & 7)) << 4)) =
            make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                       __byte_perm(v.y, v.w, 0x7632));
    }
}

template <class T, int G>
__global__ void __launch_bounds__(kW4Threads, 1) w4_rows(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ W4Params p) {
    using C = W4Cfg<G>;
    constexpr int kTokens = C::kTokens, kSub = C::kSub, kStages = C::kStages, kA = C::kA;
    extern __shared__ __align__(1024) uint8_t w4_smem[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(w4_smem) + 1023) & ~uintptr_t(1023));
    const uint32_t ring = ptx::smem_addr(smem);
    // x tiles first (1024-byte aligned swizzle atoms), then the weights (16 KB each)
    auto x_at = [&](int s) { return ring + uint32_t(s) * (kTokens * kW4StepK * 2); };
    auto w_at = [&](int s) { return ring + uint32_t(kStages * kTokens * kW4StepK * 2 + s * kW4WeightBytes); };
    uint8_t *after = smem + kStages * C::kStageBytes;
    const uint32_t bars = ptx::smem_addr(after);
    auto wfull = [&](int s) { return bars + 8u * s; };
    auto wempty = [&](int s) { return bars + 8u * (kStages + s); };
    auto xfull = [&](int s) { return bars + 8u * (2 * kStages + s); };
    auto xempty = [&](int s) { return bars + 8u * (3 * kStages + s); };
    auto afull = [&](int h, int a) { return bars + 8u * (4 * kStages + kA * h + a); };
    auto done = [&](int h, int a) { return bars + 8u * (4 * kStages + kA * (2 + h) + a); };  // A read, D written
    auto dempty = [&](int h, int d) { return bars + 8u * (4 * kStages + 4 * kA + 2 * h + d); };
    auto a_col = [&](int h, int a) { return uint32_t(64 * (kA * h + a)); };
    auto d_col = [&](int h, int d) { return uint32_t(128 * kA + C::kD * (2 * h + d)); };
    int *start = reinterpret_cast<int *>(after + C::kBars * 8);  // first row of each expert, checked
    int *first = start + kW4MaxExperts + 1;                      // token chunks of the experts before
    uint32_t *slots = reinterpret_cast<uint32_t *>(first + kW4MaxExperts + 1);
    volatile uint32_t *abort_flag = slots + 1;
    volatile int32_t *arrived = reinterpret_cast<volatile int32_t *>(slots + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(wfull(s), 1);
            ptx::mbar_init(wempty(s), 8);
            ptx::mbar_init(xfull(s), 1);
            ptx::mbar_init(xempty(s), 2);
        }
        for (int h = 0; h < 2; ++h) {
            for (int a = 0; a < kA; ++a) {
                ptx::mbar_init(afull(h, a), 4);
                ptx::mbar_init(done(h, a), 1);
            }
            for (int d = 0; d < 2; ++d)
                ptx::mbar_init(dempty(h, d), 4);
        }
        *abort_flag = 0u;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tmap(&tmap_w);
    }
    if (warp == 1) {
        ptx::tmem_alloc<1>(ptx::smem_addr(slots), 512);
        ptx::tmem_relinquish<1>();
    }
    // No wait here: w4_gather lets this kernel start when all before it has completed.
    ptx::fence_proxy_async_global();
    ptx::griddep_launch_dependents();
    const int E = p.experts;
    w4_starts(p, start);
    __syncthreads();
    {
        auto chunks_of = [&](int e) { return (max(0, start[e + 1] - start[e]) + kTokens - 1) / kTokens; };
        const int per = (E + kW4Threads - 1) / kW4Threads;
        int sum = 0;
        for (int e = tid * per; e < min(E, (tid + 1) * per); ++e)
            sum += chunks_of(e);
        int total, at = block_scan(sum, total);
        for (int e = tid * per; e < min(E, (tid + 1) * per); ++e) {
            first[e] = at;
            at += chunks_of(e);
        }
        if (tid == 0)
            first[E] = total;
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = slots[0];  // column 0: all of them are allocated
    const int64_t total = int64_t(first[E]) * p.tiles * p.steps;  // steps of the launch
    const int ctas = int(min(int64_t(gridDim.x), total));
    const int cta = blockIdx.x;
    const int64_t s_begin = cta < ctas ? total * cta / ctas : 0, s_end = cta < ctas ? total * (cta + 1) / ctas : 0;
    const Abort ab{p.status + 2, abort_flag, p.timeout_ns};
    // pieces of the range, item by item: f(item, first step, steps) in every role alike
    auto pieces = [&](auto &&f) {
        for (int64_t s = s_begin; s < s_end;) {
            const int64_t item = s / p.steps;
            const int k0 = int(s - item * p.steps), n = int(min(int64_t(p.steps - k0), s_end - s));
            f(w4_item(p, start, first, item, kTokens), item, k0, n);
            s += n;
        }
    };

    if (warp == 0) {
        const uint32_t leader = ptx::elect_one_sync();
        int st = 0;
        uint32_t ph = 0;
        bool ok = true;
        pieces([&](const W4Item &it, int64_t, int k0, int n) {
            for (int j = 0; ok && j < n; ++j) {
                ok = w4_wait(wempty(st), ph ^ 1u, ab, kStatusTimeout | kRoleProducer | uint32_t(st));
                if (!ok)
                    break;
                ptx::mbar_arrive_expect_tx(wfull(st), kW4WeightBytes, leader);
                ptx::tma_load_3d(w_at(st), &tmap_w, wfull(st), (k0 + j) * (kW4StepK / 2), it.n0, it.e, leader);
                if (++st == kStages) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        });
    } else if (warp < 3) {
        const int h = warp - 1;
        const uint32_t leader = ptx::elect_one_sync();
        int st = 0, a = 0, d = 0;
        uint32_t ph = 0, a_ph = 0, d_ph = 3;  // bits: the phases of each A's and D's next use
        bool ok = true;
        pieces([&](const W4Item &it, int64_t, int, int n) {
            const uint32_t idesc = ptx::f16_idesc(Fmt<T>::kUmma, 128, (it.count + 15) & ~15);
            const bool active = it.n0 + 128 * h < p.n;
#pragma unroll 1
            for (int j = 0; ok && j < n; ++j) {
                if (active) {
                    const bool s0 = look(xfull(st), ph), s1 = look(dempty(h, d), (d_ph >> d) & 1u);
                    ok = w4_wait(afull(h, a), (a_ph >> a) & 1u, ab, kStatusTimeout | kRoleMma | 0x40u | uint32_t(a)) &&
                         w4_wait_seen(s0, xfull(st), ph, ab, kStatusTimeout | kRoleMma | uint32_t(st)) &&
                         w4_wait_seen(s1, dempty(h, d), (d_ph >> d) & 1u, ab, kStatusTimeout | kRoleMma | 0x60u | uint32_t(d));
                    if (!ok)
                        break;
                    a_ph ^= 1u << a;
                    d_ph ^= 1u << d;
                    ptx::tc_fence_after();
                    const uint64_t bd = ptx::sw128_kmajor_desc(x_at(st));
                    w4_mma_step<G, kTokens>(d_col(h, d), a_col(h, a), uint32_t(bd), uint32_t(bd >> 32), idesc, leader);
                    ptx::umma_commit<1>(done(h, a), leader);
                } else {
                    ok = w4_wait(xfull(st), ph, ab, kStatusTimeout | kRoleMma | uint32_t(st));
                    if (!ok)
                        break;
                }
                ptx::umma_commit<1>(xempty(st), leader);
                d ^= 1;
                a = a + 1 == kA ? 0 : a + 1;
                if (++st == kStages) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        });
    } else if (warp == 3) {
        const uint32_t leader = ptx::elect_one_sync();
        int st = 0;
        uint32_t ph = 0;
        bool ok = true;
        // what precedes the launch of w4_gather is done (see there), its own writes only now
        ptx::griddep_wait();
        ptx::fence_proxy_async_global();
        pieces([&](const W4Item &it, int64_t, int k0, int n) {
            const uint32_t bytes = uint32_t(((it.count + 7) & ~7) * 256);
            const uint8_t *from = p.xs + (int64_t(it.r0 + 8 * it.e) * p.steps) * 256 + int64_t(k0) * bytes;
            for (int j = 0; ok && j < n; ++j) {
                ok = w4_wait(xempty(st), ph ^ 1u, ab, kStatusTimeout | kRoleProducer | 0x80u | uint32_t(st));
                if (!ok)
                    break;
                ptx::mbar_arrive_expect_tx(xfull(st), bytes, leader);
                bulk_load(x_at(st), from, bytes / 2, xfull(st), leader);
                bulk_load(x_at(st) + uint32_t(kTokens * 128), from + bytes / 2, bytes / 2, xfull(st), leader);
                from += bytes;
                if (++st == kStages) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        });
    } else if (warp < 12) {
        const int h = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;  // row within the half
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t w_row = uint32_t((128 * h + row) * 64) + ((uint32_t(row >> 1) & 3u) << 4);
        int st = 0, a = 0;                   // the next step's stage and A
        uint32_t ph = 0, a_ph = (1u << kA) - 1u;  // a_ph: bit a, the phase of the A's last use
        bool ok = true;
        auto next = [&]() {
            a = a + 1 == kA ? 0 : a + 1;
            if (++st == kStages) {
                st = 0;
                ph ^= 1u;
            }
        };
        pieces([&](const W4Item &it, int64_t, int k0, int n) {
            if (it.n0 + 128 * h >= p.n) {  // no columns: on with the ring
                for (int j = 0; ok && j < n; ++j) {
                    ok = w4_wait(wfull(st), ph, ab, kStatusTimeout | kRoleEpilogue | 0x80u | uint32_t(st));
                    if (ok && lane == 0)
                        ptx::mbar_arrive(wempty(st));
                    next();
                }
                return;
            }
            const uint8_t *zeros = p.zeros ? p.zeros + (int64_t(it.e) * p.n + min(it.n0 + 128 * h + row, p.n - 1)) * p.groups : nullptr;
            uint32_t ze[kSub];  // of the next step
            auto load_zeros = [&](int step) {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
                    ze[s] = zeros[kSub > 1 ? min(step * kSub + s, p.groups - 1) : step];  // past the end x is zero
            };
#pragma unroll
            for (int s = 0; s < kSub; ++s)
                ze[s] = 8u;
            if (zeros)
                load_zeros(k0);
            for (int j = 0; j < n; ++j) {
                const uint32_t a_par = (a_ph >> a) & 1u;
                const bool seen = look(done(h, a), a_par);
                ok = w4_wait(wfull(st), ph, ab, kStatusTimeout | kRoleEpilogue | 0x80u | uint32_t(st));
                if (!ok)
                    return;
                const uint32_t from = w_at(st) + w_row, to = a_col(h, a) + lanes;
                uint32_t minus[kSub];
#pragma unroll
                for (int s = 0; s < kSub; ++s)
                    minus[s] = w4_minus<T>(ze[s] & 15u);
                if (zeros && j + 1 < n)
                    load_zeros(k0 + j + 1);
                // the MMAs that read this A last are done
                ok = w4_wait_seen(seen, done(h, a), a_par, ab, kStatusTimeout | kRoleEpilogue | 0x40u | uint32_t(a));
                if (!ok)
                    return;
                ptx::tc_fence_after();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint4 v = lds128(from ^ uint32_t(c << 4));
                    const uint32_t z = minus[c * 32 / G];
                    uint32_t r[16];
                    widen<T>(v.x, z, r);
                    widen<T>(v.y, z, r + 4);
                    widen<T>(v.z, z, r + 8);
                    widen<T>(v.w, z, r + 12);
                    tmem_st_x16(to + uint32_t(16 * c), r);
                }
                tmem_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(wempty(st));
                    ptx::mbar_arrive(afull(h, a));
                }
                a_ph ^= 1u << a;
                next();
            }
        });
    } else {
        const int h = (warp - 12) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        int a = 0, d = 0;
        uint32_t a_ph = 0;
        bool ok = true;
        pieces([&](const W4Item &it, int64_t item, int k0, int n) {
            const int col = it.n0 + 128 * h + row;
            const int npad = (it.count + 15) & ~15;
            const T *scales = static_cast<const T *>(p.scales) + (int64_t(it.e) * p.n + min(col, p.n - 1)) * p.groups;
            float sum[kTokens];
#pragma unroll
            for (int i = 0; i < kTokens; ++i)
                sum[i] = 0.0f;
            // the scales are loaded two steps ahead: [0] for even steps of the piece, [1] for odd ones
            T sc[2][kSub] = {};
            auto load_scales = [&](int step, T(&v)[kSub]) {
#pragma unroll
                for (int s = 0; s < kSub; ++s)
                    v[s] = scales[kSub > 1 ? min(step * kSub + s, p.groups - 1) : step];
            };
            auto take = [&](int j, T(&v)[kSub]) {
                ok = w4_wait(done(h, a), (a_ph >> a) & 1u, ab, kStatusTimeout | kRoleEpilogue | uint32_t(a));
                if (!ok)
                    return;
                a_ph ^= 1u << a;
                ptx::tc_fence_after();
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    const float scale = to_f32(v[s]) * W4Unit<T>::kBack;
#pragma unroll
                    for (int q = 0; q < kTokens / 16; ++q)
                        if (16 * q < npad) {
                            uint32_t r[16];
                            tmem_ld_x16(d_col(h, d) + lanes + uint32_t(s * kTokens + 16 * q), r);
                            tmem_wait_ld16(r);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                sum[16 * q + i] = fmaf(scale, __uint_as_float(r[i]), sum[16 * q + i]);
                        }
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(dempty(h, d));
                if (j + 2 < n)
                    load_scales(k0 + j + 2, v);
                d ^= 1;
                a = a + 1 == kA ? 0 : a + 1;
            };
            if (it.n0 + 128 * h < p.n) {
                load_scales(k0, sc[0]);
                if (n > 1)
                    load_scales(k0 + 1, sc[1]);
                for (int j = 0; ok && j < n; j += 2) {
                    take(j, sc[0]);
                    if (ok && j + 1 < n)
                        take(j + 1, sc[1]);
                }
            } else {
                a = (a + n) % kA;
                d = (d + n) & 1;
            }
            // ---- the piece's sums: to out, or where the tile is cut to the workspace ----
            T *out = static_cast<T *>(p.out) + int64_t(it.r0) * p.n + col;
            const bool there = ok && col < p.n;
            if (n == p.steps) {
                if (there) {
#pragma unroll
                    for (int i = 0; i < kTokens; ++i)
                        if (i < it.count)
                            out[int64_t(i) * p.n] = from_f32<T>(sum[i]);
                }
                return;
            }
            const int64_t a = item * p.steps;
            const int c0 = w4_cta_of(a, total, ctas), c1 = w4_cta_of(a + p.steps - 1, total, ctas);
            // slot 0 of a CTA: a piece that begins inside its tile; slot 1: one that begins its tile
            auto slot = [&](int c) { return p.ws + int64_t(2 * c + (c == c0 ? 1 : 0)) * (kTokens * kW4TileRows) + 128 * h + row; };
            if (there) {
                float *mine = slot(cta);
#pragma unroll
                for (int i = 0; i < kTokens; ++i)
                    if (i < it.count)
                        __stcg(mine + i * kW4TileRows, sum[i]);
            }
            __threadfence();
            named_sync(2, 256);
            if (tid == 384)
                *arrived = ok ? atomicAdd(p.counters + c0, 1) : -1;
            named_sync(2, 256);
            if (*arrived != c1 - c0)
                return;
            __threadfence();
            if (tid == 384)
                p.counters[c0] = 0;
            if (there) {
                for (int i = 0; i < it.count; ++i) {
                    float s = 0.0f;
                    for (int c = c0; c <= c1; ++c)
                        s += __ldcg(slot(c) + i * kW4TileRows);
                    out[int64_t(i) * p.n] = from_f32<T>(s);
                }
            }
        });
    }

    // ---- teardown ----
    if (*abort_flag != 0u) {
        // let copies and MMAs already issued drain before the memory they target goes away
        const uint64_t t0 = ptx::globaltimer();
        while (ptx::globaltimer() - t0 < 200000ull)
            __nanosleep(1000);
        atomicCAS(p.status, 0u, *reinterpret_cast<volatile uint32_t *>(p.status + 2));
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == 1)
        ptx::tmem_dealloc<1>(tmem, 512);
}

}  // namespace moe
}  // namespace gg
