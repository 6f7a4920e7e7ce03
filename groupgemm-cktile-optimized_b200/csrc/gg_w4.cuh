// Rows in expert order times their expert's 4-bit weights with group scales, for few rows an expert:
//   out[r, n] = sum over groups g of scale[e, n, g] * sum_{k in g} (q[e, n, k] - zero[e, n, g]) x[row(r), k]
//
// What bounds it: the weights are read once, half a byte each; at HBM's rate that leaves 712 cycles an SM for a step of 256 weight
// rows x 128 k. What has to fit into them is the widening of each weight into a 16-bit operand, 9 instructions a word of 8, 5 of
// them on the ALU pipe, which starts 64 lanes a cycle (106 ns for a warp's share of a step, 32 rows: 420 of the 712 cycles), and
// the products. So each weight is widened once, whatever the number of tokens, and whatever else is on the way is kept small. Two
// forms, by how many rows an expert has (w4_few and w4_many, each explained there), share:
//
//   Work split: items (expert, token chunk, 256-row tile), cut along k where there are few, so that one token through a few experts
//   still keeps every SM reading. What is cut leaves fp32 partial sums in the workspace, which a last kernel adds in order of k.
//   w4_gather: the rows of x in expert order, laid out as the products read them, so that bulk copies load them.
#pragma once

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kW4TileRows = 256;
constexpr int kW4StepK = 128;
constexpr int kW4MaxExperts = 1024;
constexpr int kW4WeightBytes = kW4TileRows * kW4StepK / 2;  // of a step
constexpr int kW4TokenBytes = kW4StepK * 2;                 // of a token and step

struct W4Params {
    const void *x;           // [tokens or rows, k]
    const void *scales;      // [experts, n, groups]
    const uint8_t *zeros;    // [experts, n, groups] or null = 8
    const void *scales_end, *zeros_end;
    const int32_t *offsets;  // [experts + 1]
    const int32_t *src;      // [rows] slots, or null: row r reads x[r]
    void *out;               // [rows, n]
    uint32_t *status;        // [0] status word, [2] timeouts of this launch
    uint8_t *xs;             // [rows + 8 experts][steps] 256 bytes: the rows of x as the products read them (w4_gather)
    float *ws;               // partial sums: [items][splits][8][256] (w4_few), [2 x ctas][tokens of a chunk][256] (w4_many)
    int32_t *counters;       // w4_few: the next unit of work, 0 between launches
    int64_t rows, slots;     // slots: tokens * top_k
    uint64_t timeout_ns;
    int n, k, groups, experts, top_k, tiles, steps;  // steps: of 128 k
    int chunk;         // tokens of a chunk
    int ctas;          // of the product kernel
    int splits, span;  // w4_few: units of an item, steps of a unit
};

// `bytes` (a multiple of 16) from global to shared memory, counted on an mbarrier; where pred != 0.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, uint32_t pred) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar), "r"(pred)
                 : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Four bits as a 16-bit float without a conversion or a power of two to put them on: where a format's exponent field is 0 or
// 1 its value is linear in its bits, i * 2^-24 (fp16, i below 2048) and i * 2^-133 (bf16, i below 256). So a masked nibble in bits
// 0-3 or 4-7 is q or 16 q times that unit, and one fma by a power of two brings both to (q - zero) * W4Unit::kValue, exactly (the
// subnormal inputs are not flushed by it). bf16 cannot reach 1 in one multiplication, so its weights stay in units of 2^-9 (fp16's of
// 2^-12), which the fp32 sum over all groups takes back: in the scales they would carry those above 2^119 out of fp32's range. A word costs 5 instructions on the ALU pipe (one shift, four masks) and 4 on the
// FMA pipe; with powers of two or'ed in, bf16 had needed 7 and 4: 150 ns for a warp's step of 32 rows x 128 k against 111.
template <class T> struct W4Unit;
template <> struct W4Unit<__half> {
    static constexpr uint32_t kLow = 0x6c006c00u;     // 2^12: with kHigh 2^8, weights in units of 2^-12
    static constexpr uint32_t kHigh = 0x5c005c00u;    // 2^8
    static constexpr float kBack = 4096.0f;  // of a sum to its value
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
__device__ __forceinline__ bool w4_wait_slow(uint32_t bar, uint32_t parity, const Abort ab, uint32_t code) {
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

// A launch's work as one CTA sees it: items in expert order, an item's steps in order of k, and this CTA's range of steps.
struct W4Item {
    int e, n0, r0, count;
};
struct W4Work {
    const int *start, *first;  // shared: first row of each expert (checked), token chunks of the experts before
    int64_t total, begin, end;  // steps: of the launch, this CTA's range
    int ctas;

    // offsets come from the device: each is held to the range that the rows allow. Returns whether they fall anywhere; then no expert gets
    // rows: what is sized by the rows (items, workspace, 32-bit indices) holds for rising offsets. By all threads of the block, which are
    // together after it. (Setting start to 0 here in place of a flag cost one token's products 0.6 us of 36.)
    static __device__ __forceinline__ bool starts(const W4Params &p, int *start) {
        bool falls = false;
        for (int e = threadIdx.x; e <= p.experts; e += blockDim.x) {
            const int64_t v = p.offsets[e], before = e ? p.offsets[e - 1] : 0;
            falls |= v < before;
            if (v < before || v > p.rows)
                report(p.status, kSiteOffsets);
            start[e] = int(max(int64_t(0), min(v, p.rows)));
        }
        return __syncthreads_or(falls) != 0;
    }
    __device__ __forceinline__ W4Work(const W4Params &p, int *start_, int *first_) : start(start_), first(first_) {
        const int E = p.experts, tid = threadIdx.x;
        const bool falls = starts(p, start_);
        auto chunks_of = [&](int e) { return (start[e + 1] - start[e] + p.chunk - 1) / p.chunk; };
        const int per = (E + int(blockDim.x) - 1) / int(blockDim.x);
        int sum = 0, chunks;
        for (int e = tid * per; e < min(E, (tid + 1) * per); ++e)
            sum += chunks_of(e);
        int at = block_scan(sum, chunks);
        for (int e = tid * per; e < min(E, (tid + 1) * per); ++e) {
            first_[e] = at;
            at += chunks_of(e);
        }
        if (tid == 0)
            first_[E] = falls ? 0 : chunks;
        __syncthreads();
        total = int64_t(falls ? 0 : chunks) * p.tiles * p.steps;
        ctas = int(min(int64_t(p.ctas), total));
        const int cta = blockIdx.x;
        begin = cta < ctas ? total * cta / ctas : 0;
        end = cta < ctas ? total * (cta + 1) / ctas : 0;
    }
    __device__ __forceinline__ W4Item at(const W4Params &p, int item) const {
        const int run = item / p.tiles;  // token chunk of the launch, were a chunk's tiles in a row
        int lo = 0, hi = p.experts - 1;  // the last expert whose first chunk is at or before it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= run)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int chunks = first[lo + 1] - first[lo], in = item - first[lo] * p.tiles;
        const int tile = in / chunks, chunk = in - tile * chunks;
        const int r0 = start[lo] + chunk * p.chunk;
        return {lo, tile * kW4TileRows, r0, min(p.chunk, start[lo + 1] - r0)};
    }
    // The range's pieces, item by item, alike in every warp: f(place of the item, its number, first step, steps).
    template <class F> __device__ __forceinline__ void pieces(const W4Params &p, F &&f) const {
        for (int64_t s = begin; s < end;) {
            const int64_t item = s / p.steps;
            const int k0 = int(s - item * p.steps), n = int(min(int64_t(p.steps - k0), end - s));
            f(at(p, int(item)), item, k0, n);
            s += n;
        }
    }
    __device__ __forceinline__ int cta_of(int64_t step) const { return int(((step + 1) * ctas - 1) / total); }
    __device__ __forceinline__ int first_cta(const W4Params &p, int64_t item) const { return cta_of(item * p.steps); }
    __device__ __forceinline__ int last_cta(const W4Params &p, int64_t item) const { return cta_of(item * p.steps + p.steps - 1); }
    // Partial sums [token][256] of CTA c's piece of a cut item: slot 0 where the piece begins inside its tile, 1 where it begins it.
    __device__ __forceinline__ float *slot(const W4Params &p, int c, int first_of_item) const {
        return p.ws + int64_t(2 * c + (c == first_of_item ? 1 : 0)) * (p.chunk * kW4TileRows);
    }
};

// The rows of x in expert order, gathered through src, as the products read them: for each chunk of an expert's tokens and each
// step of 128 k, pieces of eight values in the order in which masks and shifts take the weights out of a word, placed
//   kFragments: as mma.sync's B fragments of 8 tokens (a word of k after another, 16 bytes a lane),
//   else:       as a shared-memory image of tcgen05's B (K-major, two halves of 64 k, each a row of 128 bytes a token with the
//               128-byte swizzle).
// Token count rounded up to 8: what the places of the missing tokens hold goes into columns that nothing reads. (Done by warps of the product kernel instead, with cp.async and shared memory, this took them 1400 cycles a step
// at 16 tokens: twice what HBM allows.) Rows of no expert are set to zero in out.
constexpr int kW4GatherThreads = 128;
template <class T, bool kFragments> __global__ void __launch_bounds__(kW4GatherThreads) w4_gather(const __grid_constant__ W4Params p) {
    __shared__ int start[kW4MaxExperts + 1];
    ptx::griddep_wait();
    // The product kernel may start now. It reads what earlier kernels wrote (offsets, scales, weights) without waiting for this one
    // to end: every block of this one has passed its own wait by then. Before it reads xs it waits for this one.
    ptx::griddep_launch_dependents();
    const bool falls = W4Work::starts(p, start);
    const int pieces = p.steps * (kW4StepK / 8), first_piece = int(blockIdx.y) * kW4GatherThreads + int(threadIdx.x);
    const int more = int(gridDim.y) * kW4GatherThreads;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        if (falls || r < start[0] || r >= start[p.experts]) {
            for (int col = first_piece; col < p.n; col += more)
                static_cast<T *>(p.out)[r * p.n + col] = from_f32<T>(0.0f);
            continue;
        }
        int64_t row = r;
        if (p.src) {
            const int s = p.src[r];
            row = s < 0 || s >= p.slots ? -1 : s / p.top_k;
            if (row < 0 && first_piece == 0)
                report(p.status, kSiteSrc);
        }
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
        const T *from = static_cast<const T *>(p.x) + row * p.k;
        uint8_t *to = p.xs + int64_t(int(r) - i + 8 * lo) * p.steps * kW4TokenBytes;
#pragma unroll 4
        for (int piece = first_piece; piece < pieces; piece += more) {
            const int step = piece >> 4, c = piece & 15;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row >= 0 && piece * 8 < p.k)
                v = __ldg(reinterpret_cast<const uint4 *>(from + piece * 8));
            const int at = kFragments ? (((i >> 3) * 4 + (c >> 2)) * 32 + (i & 7) * 4 + (c & 3)) * 16
                                      : ((c >> 3) * count + i) * 128 + (((c & 7) ^ (i & 7)) << 4);
            *reinterpret_cast<uint4 *>(to + int64_t(step) * count * kW4TokenBytes + at) =
                make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                           __byte_perm(v.y, v.w, 0x7632));
        }
    }
}

// ---- few rows an expert: chunks of 8 tokens, mma.sync ----
//
// The words of weights that ldmatrix hands to a lane are those of its place in the A fragment, so they are widened in the
// registers that mma.sync reads, and nothing but a wait and an arrival stands between a step's bytes and its products. 8 warps of 32
// weight rows and a loading warp (a TMA box of weights, a bulk copy of tokens a step, a ring of 4 steps), two CTAs an SM. Units
// of work are taken from a counter, so that CTAs that share an SM with a slower one do not wait for it at the end.
// Measured: 8 experts of 4096 x 7168 (117 MB of weights) in groups of 128, 1 row each, 35.3 us, and 24.5 us for each further 117 MB
// (4.8 TB/s, 73% of the measured copy rate): the rest is the start of three launches, the first loads and the sum of split items.
// 8 rows each 39.4. Above that an expert's weights are widened again for each 8 tokens; in one pass mma.sync's own rate binds (11
// cycles an instruction and scheduler: 16 tokens 36 us for each further 117 MB).
constexpr int kW4FewTokens = 8;
constexpr int kW4FewThreads = kW4TileRows + 32;
constexpr int kW4FewUnits = 4;  // units of work a CTA, where items have to be split for that
constexpr int kW4FewRing = 8;   // units that the loading warp may be ahead: stages and two
constexpr int kW4FewStages = 4;
constexpr int kW4FewSmem = 1024 + kW4FewStages * (kW4WeightBytes + kW4FewTokens * kW4TokenBytes);

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), 16-bit operands.
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with zero for D's old values.
template <class T>
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Four 8 x 16-byte matrices; lane l gets word l % 4 of row l / 4 of each.
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Eight values of kBytes each (a scale or a zero of a group each) of a row as a queue of 32-bit words, and the next eight on
// the way. Where rows are a multiple of eight groups long a visit is one load at a multiple of eight; else a row starts at
// any multiple of kBytes and a visit is its words one by one. The lanes' rows lie in lines of their own, so each load costs a
// warp 32 visits to L1, and five a visit instead of one showed: 37 tokens x 4 of 32 experts of 7168 x 2048 in groups of 64 with
// zeros took 73.4 us against 69.6, 8 experts of 4096 x 7168 in groups of 128 0.5 to 1 us of 36 to 51.
template <int kBytes> struct W4Queue {
    static constexpr int kWords = 2 * kBytes;  // of eight values
    const uint32_t *from;                      // the aligned word that holds the next visit's first value
    const uint32_t *end;                       // past the array's last word
    int at;                                    // that visit's first group
    int drop;                                  // its values before the first one asked for
    uint32_t shift;                            // bits from the word's start to the value
    uint32_t raw[kWords + 1], word[kWords];

    // From now on the values from `first` on of a row of `groups`: the visit is on its way, to be taken by the next refill.
    __device__ __forceinline__ void begin(const void *array, int64_t row, int groups, const void *array_end, int first) {
        drop = groups % 8 == 0 ? first & 7 : 0;
        at = first - drop;
        const uintptr_t p = reinterpret_cast<uintptr_t>(array) + uintptr_t((row * groups + at) * kBytes);
        from = reinterpret_cast<const uint32_t *>(p & ~uintptr_t(3));
        shift = uint32_t(p & 3) * 8;
        end = static_cast<const uint32_t *>(array_end);
        load(groups);
    }
    __device__ __forceinline__ void load(int groups) {
        if (groups % 8 == 0) {
            if constexpr (kBytes == 2) {
                const uint4 v = __ldg(reinterpret_cast<const uint4 *>(from));
                raw[0] = v.x, raw[1] = v.y, raw[2] = v.z, raw[3] = v.w;
            } else {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(from));
                raw[0] = v.x, raw[1] = v.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i <= kWords; ++i)
                raw[i] = from + i < end ? __ldg(from + i) : 0u;
        }
        from += kWords;
    }
    // Up to eight values into the queue (returned: how many), and the next visit on its way where there is one before group `last`.
    // Past the row's last group the values are 0: the sums of a step's groups there are 0, and the next row's scale may be infinite or NaN.
    __device__ __forceinline__ int refill(int groups, int last) {
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            word[i] = __funnelshift_r(raw[i], raw[i + 1], shift);
        const int left = groups - at;
        if (left < 8) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const int bits = 8 * (left * kBytes - 4 * i);  // of this word, inside the row
                word[i] = bits >= 32 ? word[i] : bits > 0 ? word[i] & ((1u << bits) - 1u) : 0u;
            }
        }
        at += 8;
        if (at < last)
            load(groups);
        const int values = 8 - drop;
        for (; drop > 0; --drop)
            take();
        return values;
    }
    __device__ __forceinline__ uint32_t take() {
        const uint32_t v = word[0] & ((1u << (8 * kBytes)) - 1u);
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            word[i] = __funnelshift_r(word[i], i + 1 < kWords ? word[i + 1] : 0u, 8 * kBytes);
        return v;
    }
};

// Items of the launch.
__device__ __forceinline__ int w4_items(const W4Params &p, const int *first) { return first[p.experts] * p.tiles; }
// A unit's sums [token][256], where items are split.
__device__ __forceinline__ float *w4_sums(const W4Params &p, int item, int split) {
    return p.ws + (int64_t(item) * p.splits + split) * (kW4FewTokens * kW4TileRows);
}

// Adds the sums of split items, in order of k. A kernel of its own: joined inside w4_few, by the last unit of an item to arrive, each
// arrival's fence waited some microseconds behind the streaming weights, and one unit more a CTA cost as much.
template <class T> __global__ void __launch_bounds__(kW4TileRows) w4_add(const __grid_constant__ W4Params p) {
    __shared__ int start[kW4MaxExperts + 1], first[kW4MaxExperts + 1];
    ptx::griddep_launch_dependents();
    const W4Work work(p, start, first);  // the offsets are older than w4_few
    const int items = w4_items(p, first), t = threadIdx.x;
    bool waited = false;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const W4Item it = work.at(p, item);
        if (!waited)
            ptx::griddep_wait();
        waited = true;
        float v[kW4FewTokens] = {};
#pragma unroll 4
        for (int split = 0; split < p.splits; ++split)
#pragma unroll
            for (int u = 0; u < kW4FewTokens; ++u)
                if (u < it.count)
                    v[u] += __ldcg(w4_sums(p, item, split) + u * kW4TileRows + t);
        if (it.n0 + t >= p.n)
            continue;
#pragma unroll
        for (int u = 0; u < kW4FewTokens; ++u)
            if (u < it.count)
                static_cast<T *>(p.out)[int64_t(it.r0 + u) * p.n + it.n0 + t] = from_f32<T>(v[u]);
    }
    if (!waited)
        ptx::griddep_wait();  // this kernel ends after w4_few
}

template <class T, int G, bool kZeros>
__global__ void __launch_bounds__(kW4FewThreads, 2) w4_few(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ W4Params p) {
    constexpr int kSub = kW4StepK / G;  // groups a step
    constexpr int kXBytes = kW4FewTokens * kW4TokenBytes;
    extern __shared__ __align__(1024) uint8_t w4_smem[];
    __shared__ int start[kW4MaxExperts + 1], first[kW4MaxExperts + 1];
    __shared__ uint64_t bar_words[2 * kW4FewStages + 1];
    struct Unit {
        W4Item it;
        int item, split, k0, n;  // n: steps; 0: no more units
    };
    __shared__ Unit ring[kW4FewRing];  // the CTA's units, each there before the last eight groups of the one before it are
    __shared__ uint32_t abort_word;
    volatile uint32_t *abort_flag = &abort_word;
    const uint32_t smem = (ptx::smem_addr(w4_smem) + 1023) & ~1023u, bars = ptx::smem_addr(bar_words);
    auto w_at = [&](int s) { return smem + uint32_t(s * kW4WeightBytes); };
    auto x_at = [&](int s) { return smem + uint32_t(kW4FewStages * kW4WeightBytes + s * kXBytes); };
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kW4FewStages + s); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int s = 0; s < kW4FewStages; ++s) {
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), 8);
        }
        ptx::mbar_init(bars + 8u * (2 * kW4FewStages), 1);
        *abort_flag = 0u;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tmap(&tmap_w);
    }
    // No wait here: w4_gather lets this kernel start when all before it has completed.
    ptx::fence_proxy_async_global();
    ptx::griddep_launch_dependents();
    const W4Work work(p, start, first);
    const int items = w4_items(p, first), units = items * p.splits, ctas = min(int(gridDim.x), units);
    const Abort ab{p.status + 2, abort_flag, p.timeout_ns};
    int st = 0;
    uint32_t ph = 0;
    auto next = [&]() {
        if (++st == kW4FewStages) {
            st = 0;
            ph ^= 1u;
        }
    };
    bool ok = true;
    if (warp == 8) {
        const uint32_t leader = ptx::elect_one_sync();
        auto publish = [&](int seq, int u) {
            Unit r{};
            if (u < units) {
                r.item = u / p.splits;
                r.split = u - r.item * p.splits;
                r.k0 = r.split * p.span;
                r.n = min(p.span, p.steps - r.k0);
                r.it = work.at(p, r.item);
            }
            if (leader)
                ring[seq % kW4FewRing] = r;
            return r;
        };
        bool gathered = false;
        auto ask = [&]() {  // for the CTA's next unit; the last of the launch's askers puts the counter back
            int v = 0;
            if (lane == 0) {
                v = atomicAdd(p.counters, 1);
                if (v == units - 1)
                    *p.counters = 0;
            }
            return v;
        };
        Unit r = publish(0, int(blockIdx.x));
        int asked = r.n > 0 ? ask() : 0;
        ptx::mbar_arrive_expect_tx(bars + 8u * (2 * kW4FewStages), 0, leader);  // the first unit is there
        for (int seq = 1; ok && r.n > 0; ++seq) {
            Unit after{};
            const uint8_t *from = p.xs + (int64_t(r.it.r0 + 8 * r.it.e) * p.steps + int64_t(r.k0) * kW4FewTokens) * kW4TokenBytes;
            auto weights = [&](int j) {
                if (j == max(0, r.n - 8 / kSub)) {  // before the consumers' last visit to this unit's scales
                    after = publish(seq, ctas + __shfl_sync(0xffffffffu, asked, 0));
                    if (after.n > 0)
                        asked = ask();
                }
                ptx::mbar_arrive_expect_tx(full(st), kW4WeightBytes + kXBytes, leader);
                ptx::tma_load_3d(w_at(st), &tmap_w, full(st), (r.k0 + j) * (kW4StepK / 2), r.it.n0, r.it.e, leader);
            };
            auto tokens = [&](int j, int s) { bulk_load(x_at(s), from + j * kXBytes, kXBytes, full(s), leader); };
            int j = 0;
            if (!gathered) {
                // What precedes the launch of w4_gather is done (see there), its own writes only after this wait: the first steps' weights
                // are asked for before it.
                const int ahead = min(kW4FewStages, r.n);
                for (; j < ahead; ++j) {
                    weights(j);
                    next();
                }
                ptx::griddep_wait();
                ptx::fence_proxy_async_global();
                for (int i = 0; i < ahead; ++i)
                    tokens(i, i);
                gathered = true;
            }
            for (; ok && j < r.n; ++j) {
                ok = w4_wait(empty(st), ph ^ 1u, ab, kStatusTimeout | kRoleProducer | uint32_t(st));
                if (!ok)
                    break;
                weights(j);
                tokens(j, st);
                next();
            }
            r = after;
        }
        if (!gathered)
            ptx::griddep_wait();  // this kernel ends after w4_gather
    } else {
        // of ldmatrix: row lane % 8 of the warp's, piece lane / 8 swizzled
        const uint32_t w_lane = uint32_t((warp * 32 + (lane & 7)) * 64) + (uint32_t((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
        // Scales and zeros of weight row `lane`, to be handed to the lanes whose fragments hold the row.
        W4Queue<2> scales;
        W4Queue<1> zeros;
        auto begin = [&](const Unit &r) {
            const int64_t row = int64_t(r.it.e) * p.n + min(r.it.n0 + warp * 32 + lane, p.n - 1);
            scales.begin(p.scales, row, p.groups, p.scales_end, r.k0 * kSub);
            if constexpr (kZeros)
                zeros.begin(p.zeros, row, p.groups, p.zeros_end, r.k0 * kSub);
        };
        ok = w4_wait(bars + 8u * (2 * kW4FewStages), 0, ab, kStatusTimeout | kRoleMma | 0x80u);
        Unit r{};
        if (ok)
            r = ring[0];
        if (r.n > 0)
            begin(r);
        for (int seq = 1; ok && r.n > 0; ++seq) {
            float sum[2][4] = {};
            int queued = 0;  // groups in the queues
            for (int j = 0; j < r.n; ++j) {
                ok = w4_wait(full(st), ph, ab, kStatusTimeout | kRoleMma | uint32_t(st));
                if (!ok)
                    break;
                if (queued == 0) {
                    queued = scales.refill(p.groups, (r.k0 + r.n) * kSub);
                    if constexpr (kZeros)
                        zeros.refill(p.groups, (r.k0 + r.n) * kSub);
                    if (scales.at >= (r.k0 + r.n) * kSub) {  // this unit's last visit: the next one's scales are on their way from here
                        const Unit after = ring[seq % kW4FewRing];
                        if (after.n > 0)
                            begin(after);
                    }
                }
                queued -= kSub;
                uint32_t w[4][4];  // rows g + 8 i; word c holds k = 32 c + 8 t ...
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    ldmatrix_x4(w_at(st) + w_lane + uint32_t(i * 512), w[i]);
                const uint32_t x_from = x_at(st) + uint32_t(lane * 16);
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    float acc[2][4];
                    uint32_t minus[4];
                    if constexpr (kZeros) {
                        const uint32_t mine = w4_minus<T>(zeros.take() & 15u);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            minus[i] = __shfl_sync(0xffffffffu, mine, g + 8 * i);
                    } else {
                        minus[0] = minus[1] = minus[2] = minus[3] = w4_minus<T>(8u);
                    }
#pragma unroll
                    for (int c = s * 4 / kSub; c < (s + 1) * 4 / kSub; ++c) {
                        uint32_t a[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            widen<T>(w[i][c], minus[i], a[i]);
                        const uint4 b = lds128(x_from + uint32_t(c * 512));
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            if (c == s * 4 / kSub)
                                mma16816_first<T>(acc[m], a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b.x, b.y);
                            else
                                mma16816<T>(acc[m], a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b.x, b.y);
                            mma16816<T>(acc[m], a[2 * m][2], a[2 * m + 1][2], a[2 * m][3], a[2 * m + 1][3], b.z, b.w);
                        }
                    }
                    if (s == kSub - 1) {
                        // All of the stage is in registers. TMA writes it next: the lanes' reads are ordered before that by the
                        // proxy fence (without it, reads still on the way met the next step's bytes).
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0)
                            ptx::mbar_arrive(empty(st));
                    }
                    const uint16_t bits = uint16_t(scales.take());
                    const float scale = to_f32(*reinterpret_cast<const T *>(&bits));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = __shfl_sync(0xffffffffu, scale, g + 8 * i);
                        float *to = sum[i >> 1] + 2 * (i & 1);
                        to[0] = fmaf(f, acc[i >> 1][2 * (i & 1)], to[0]);
                        to[1] = fmaf(f, acc[i >> 1][2 * (i & 1) + 1], to[1]);
                    }
                }
                next();
            }
            if (!ok)
                break;
            const W4Item &it = r.it;
            T *out = static_cast<T *>(p.out) + int64_t(it.r0) * p.n + it.n0 + warp * 32;
            float *mine = w4_sums(p, r.item, r.split) + warp * 32;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * m + 8 * (i >> 1) + g, tok = 2 * t + (i & 1);
                    if (tok >= it.count || it.n0 + warp * 32 + row >= p.n)
                        continue;
                    const float v = sum[m][i] * W4Unit<T>::kBack;
                    if (p.splits == 1)
                        out[int64_t(tok) * p.n + row] = from_f32<T>(v);
                    else
                        __stcg(mine + tok * kW4TileRows + row, v);
                }
            r = ring[seq % kW4FewRing];
        }
    }
    if (*abort_flag != 0u) {
        // let copies already asked for drain before the memory they target goes away
        const uint64_t t0 = ptx::globaltimer();
        while (ptx::globaltimer() - t0 < 200000ull)
            __nanosleep(1000);
        atomicCAS(p.status, 0u, *reinterpret_cast<volatile uint32_t *>(p.status + 2));
    }
}

// ---- more rows an expert: chunks of up to 32 tokens, tcgen05 ----
//
//   warp 0       TMA: a step's weights into a ring of 6 steps
//   warp 3       bulk copies of a step's tokens
//   warps 4-11   a group of four for each half of the weight rows, a thread a row: 16 bytes at a time from the ring,
//                widened in registers, tcgen05.st into the half's next A operand
//   warps 1, 2   a half each: tcgen05.mma, D[weight row, token] = A (Tensor Memory) x B (tokens), a fresh accumulator
//                a group
//   warps 12-19  a half each four: tcgen05.ld of a step's products and the fp32 sum with the group's scale (one scalar a
//                thread); output
//
// Three A operands and two D a half keep the widening from waiting for the MMAs. Measured: 8 experts of 4096 x 7168 (117 MB of
// weights) in groups of 128, 8 rows each, 50.4 us, 16 51.1, 32 53.9, and 29.8, 29.8 and 32.9 us for each further 117 MB. No one part binds it (31 at the time):
// without the widening 26, without that and tcgen05.st 24, without the products 27, without the sums 28, with all weights from L2 30;
// the parts share the schedulers' issue slots (3000 instructions a step and SM, 1200 of them widening). Four warps that
// issue the products in place of two gained 1 us at 8 rows and none at 32; eight more widening warps lost 3. Long runs of the
// largest sizes meet the power cap: 128 tokens x 8 of 64 experts take 300 us in 100 calls and 326 in 3000.
constexpr int kW4ManyThreads = 640;

// Tokens of a chunk: at most 32 (a thread holds a sum a token). Tensor Memory's 512 columns hold for each half kA operands of
// 64 columns and two D of a column a token and group of a step.
template <int G> struct W4Many {
    static constexpr int kSub = kW4StepK / G;  // groups a step
    static constexpr int kTokens = kSub == 4 ? 16 : 32;
    static constexpr int kA = kSub == 1 ? 3 : 2;
    static constexpr int kD = kSub * kTokens;  // columns of a D
    static constexpr int kStageBytes = kW4WeightBytes + kTokens * kW4StepK * 2;
    static constexpr int kStages = 6;  // a multiple of 2 and of kA: a stage always meets the same D and A
    static constexpr int kBars = 4 * kStages + 4 * kA + 4;
    static_assert(2 * (64 * kA + 2 * kD) <= 512 && kStages % kA == 0 && kStages % 2 == 0, "Tensor Memory");
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kBars * 8 + 64;
};

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
template <class T, int G>
__global__ void __launch_bounds__(kW4ManyThreads, 1) w4_many(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ W4Params p) {
    using C = W4Many<G>;
    constexpr int kTokens = C::kTokens, kSub = C::kSub, kStages = C::kStages, kA = C::kA;
    extern __shared__ __align__(1024) uint8_t w4_smem[];
    __shared__ int start[kW4MaxExperts + 1], first[kW4MaxExperts + 1];
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
    uint32_t *slots = reinterpret_cast<uint32_t *>(after + C::kBars * 8);
    volatile uint32_t *abort_flag = slots + 1;
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
    const W4Work work(p, start, first);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = slots[0];  // column 0: all of them are allocated
    const Abort ab{p.status + 2, abort_flag, p.timeout_ns};
    if (warp == 0) {
        const uint32_t leader = ptx::elect_one_sync();
        int st = 0;
        uint32_t ph = 0;
        bool ok = true;
        work.pieces(p, [&](const W4Item &it, int64_t, int k0, int n) {
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
        work.pieces(p, [&](const W4Item &it, int64_t, int, int n) {
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
        work.pieces(p, [&](const W4Item &it, int64_t, int k0, int n) {
            const uint32_t bytes = uint32_t(((it.count + 7) & ~7) * 256);
            const uint8_t *from = p.xs + (int64_t(it.r0 + 8 * it.e) * p.steps) * kW4TokenBytes + int64_t(k0) * bytes;
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
        work.pieces(p, [&](const W4Item &it, int64_t, int k0, int n) {
            if (it.n0 + 128 * h >= p.n) {  // no columns: on with the ring
                for (int j = 0; ok && j < n; ++j) {
                    ok = w4_wait(wfull(st), ph, ab, kStatusTimeout | kRoleEpilogue | 0x80u | uint32_t(st));
                    if (ok && lane == 0)
                        ptx::mbar_arrive(wempty(st));
                    next();
                }
                return;
            }
            W4Queue<1> zeros;
            int queued = 0;  // groups in it
            if (p.zeros)
                zeros.begin(p.zeros, int64_t(it.e) * p.n + min(it.n0 + 128 * h + row, p.n - 1), p.groups, p.zeros_end, k0 * kSub);
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
                    minus[s] = w4_minus<T>(8u);
                if (p.zeros) {
                    if (queued == 0)
                        queued = zeros.refill(p.groups, (k0 + n) * kSub);
                    queued -= kSub;
#pragma unroll
                    for (int s = 0; s < kSub; ++s)
                        minus[s] = w4_minus<T>(zeros.take() & 15u);
                }
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
        work.pieces(p, [&](const W4Item &it, int64_t item, int k0, int n) {
            const int col = it.n0 + 128 * h + row;
            const int npad = (it.count + 15) & ~15;
            float sum[kTokens];
#pragma unroll
            for (int i = 0; i < kTokens; ++i)
                sum[i] = 0.0f;
            W4Queue<2> scales;
            int queued = 0;  // groups in it
            auto take = [&]() {
                ok = w4_wait(done(h, a), (a_ph >> a) & 1u, ab, kStatusTimeout | kRoleEpilogue | uint32_t(a));
                if (!ok)
                    return;
                a_ph ^= 1u << a;
                ptx::tc_fence_after();
#pragma unroll
                for (int s = 0; s < kSub; ++s) {
                    const uint16_t bits = uint16_t(scales.take());
                    const float scale = to_f32(*reinterpret_cast<const T *>(&bits));
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
                d ^= 1;
                a = a + 1 == kA ? 0 : a + 1;
            };
            if (it.n0 + 128 * h < p.n) {
                scales.begin(p.scales, int64_t(it.e) * p.n + min(col, p.n - 1), p.groups, p.scales_end, k0 * kSub);
                for (int j = 0; ok && j < n; ++j) {
                    if (queued == 0)
                        queued = scales.refill(p.groups, (k0 + n) * kSub);
                    queued -= kSub;
                    take();
                }
            } else {
                a = (a + n) % kA;
                d = (d + n) & 1;
            }
            const bool whole = n == p.steps;
            if (!ok || col >= p.n)
                return;
            if (whole) {
                T *out = static_cast<T *>(p.out) + int64_t(it.r0) * p.n + col;
#pragma unroll
                for (int i = 0; i < kTokens; ++i)
                    if (i < it.count)
                        out[int64_t(i) * p.n] = from_f32<T>(sum[i] * W4Unit<T>::kBack);
            } else {
                float *mine = work.slot(p, blockIdx.x, work.first_cta(p, item)) + 128 * h + row;
#pragma unroll
                for (int i = 0; i < kTokens; ++i)
                    if (i < it.count)
                        __stcg(mine + i * kW4TileRows, sum[i] * W4Unit<T>::kBack);
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

// Adds the partial sums of the tiles that w4_many's ranges cut, in order of k: block c those of the tile in which CTA c's range begins
// after the CTA before has begun it, eight tokens a row of blocks. (Inside w4_many, by the last to arrive, fence, arrival and sum
// took 5 us and more with the tokens.)
template <class T> __global__ void __launch_bounds__(kW4TileRows) w4_join(const __grid_constant__ W4Params p) {
    __shared__ int start[kW4MaxExperts + 1], first[kW4MaxExperts + 1];
    ptx::griddep_launch_dependents();
    const W4Work work(p, start, first);  // the offsets are older than w4_many
    const int64_t item = work.begin / p.steps;
    const int c = blockIdx.x, u0 = int(blockIdx.y) * 8, t = threadIdx.x;
    const bool cut = work.begin < work.end && work.begin % p.steps != 0 && work.first_cta(p, item) == c - 1;
    ptx::griddep_wait();
    if (!cut)
        return;
    const W4Item it = work.at(p, int(item));
    if (it.n0 + t >= p.n)
        return;
    float v[8] = {};
    const int last = work.last_cta(p, item);
#pragma unroll 2
    for (int i = c - 1; i <= last; ++i) {
        const float *from = work.slot(p, i, c - 1) + t;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (u0 + u < it.count)
                v[u] += __ldcg(from + (u0 + u) * kW4TileRows);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
        if (u0 + u < it.count)
            static_cast<T *>(p.out)[int64_t(it.r0 + u0 + u) * p.n + it.n0 + t] = from_f32<T>(v[u]);
}

}  // namespace moe
}  // namespace gg
