// Rows in expert order times their expert's 8-bit weights, with a scale a row and a scale a weight row:
//   out[r, n] = x_scales[row(r)] * scales[e, n] * sum_k x[row(r), k] w[e, n, k]
//
// The sums are whole numbers, exact in 32 bits (k <= kI8MaxK), so neither how the work is cut nor who adds up changes a result.
//
// tcgen05.mma kind::i8 on CTA pairs, the weights as A (256 rows a pair) and a chunk of tokens as B, as wide as the chunk has tokens
// (32 to 256 in steps of 32): few rows an expert cost the bytes of its weights and next to no products, many rows run at the full
// tile, and nothing is padded to a tile of tokens.
//
//   i8_rows: the rows of x in expert order, rounded to 8 bits where they come in 16. (TMA gathers of four rows in the product kernel
//   would spare it, but take 44 cycles each: a stage of 128 rows a CTA 1400 cycles, of which the products need 512.)
//   i8_products. Work split: items (expert, token chunk, 256 weight rows). Each pair takes whole items in turn; where it pays (i8_cuts), the
//   items that would leave pairs idle at the end (or all, where there are few) are cut along k into equal ranges of steps, one a pair, taken first. What is cut
//   leaves its sums in the workspace, and the last warp to arrive adds them up (no order to keep).
//   Warps: 0 loads (weights and tokens, a ring of stages), 1 issues the products (of the pair's first CTA), 2-9 take the sums out of
//   Tensor Memory, two accumulators in turn.
// What bounds it: few rows, the weights' bytes (64 experts of 4096 x 7168, 16 rows each on average: 271 us alone, 6.9 TB/s; one token through 8 of
// them 42 us with the rows before, of which 36 are bytes); many, the tensor pipe (8 experts of 4096 rows: 557-573 us, 3.4 POPS, 93-95% of its cycles) and,
// where calls follow one another, the power cap.
#pragma once

#include "gg_moe.cuh"
#include "gg_norm.cuh"

namespace gg {
namespace moe {

constexpr int kI8TileRows = 256;    // weight rows of a pair's tile
constexpr int kI8StepK = 128;       // bytes of k of a stage: a swizzle atom's row
constexpr int kI8MaxTokens = 256;   // of a chunk
constexpr int kI8MaxExperts = 1024;
constexpr int kI8MaxK = 131056;     // k * 128 * 128 stays below 2^31
constexpr int kI8WeightBytes = 128 * kI8StepK;  // of a CTA and stage
constexpr int kI8MaxStages = 12;
constexpr int kI8Ring = 192 * 1024;
constexpr int kI8EpilogueWarps = 8;
constexpr int kI8Threads = (2 + kI8EpilogueWarps) * 32;
constexpr int kI8Smem = kI8Ring + 1024;
// Of a cut piece, at least. It counts where cut items have fewer steps than 16 for each pair; us with 4 / 8 / 16 / 32 for 20 rows of one expert of
// 2048 x 4096 13.1 / 12.1 / 13.0 / 13.9, 1000 x 8192 15.5 / 13.5 / 13.8 / 16.1, 512 x 7168 14.1 / 12.7 / 14.0 / 17.0, 1024 x 16384 19.1 / 16.8 / 15.3 / 17.0.
constexpr int kI8MinSteps = 16;
constexpr int kI8Band = 8;          // tiles whose weights are visited together (see I8Cursor)

struct I8Params {
    const void *x;            // [tokens or rows, k], as the caller has them (i8_rows)
    const float *x_scales;    // [tokens or rows], or null: x is in 16 bits (i8_rows)
    int8_t *xq;               // [rows, k] in expert order
    float *xq_scales;         // [rows]
    const float *scales;      // [experts, n]
    const int32_t *offsets;   // [experts + 1]
    const int32_t *src;       // [rows] slots, or null: row r is x[r]
    int32_t *inv;             // [slots] places (i8_token_rows)
    void *out;                // [rows, n]
    uint32_t *status;         // [0] status word, [2] timeouts of this launch
    int32_t *ws;              // [2 x pairs][2 CTAs][4 quarters][chunk / 16][4][32] int4
    int32_t *counters;        // [pairs][2 CTAs][8 warps], 0 between launches
    int64_t rows, slots;      // slots: tokens * top_k
    uint64_t timeout_ns;
    int n, k, experts, top_k, tiles, steps;
    int chunk;                // most tokens of a chunk, a multiple of 32
    int test_stall;           // test only: 1 = the first pair's first stage waits for an arrival that never comes
    int stages, stage_bytes;
    // 1: i8_rows precedes. Everything before that is done when this kernel starts, for i8_rows' blocks have waited for it, but this kernel has not
    // itself: what it reads before its own wait (offsets; weights, by TMA) comes from L2, not from what an SM may still hold of an earlier run.
    int after_rows;
};

// Instruction descriptor of kind::i8: D s32 (2 at bit 4), A and B signed (1 at bits 7 and 10), both K-major, N >> 3, M >> 4.
__host__ __device__ constexpr uint32_t i8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t pred) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(pred)
                 : "memory");
}

// Whether the items that do not fill a last round of the pairs are cut along k. What it saves: of wide chunks, which the products bind, the part
// of a round that pairs would be idle; of narrow ones, which memory binds, the part below about half, since fewer pairs at work load faster. What
// it costs, in steps, grows with the sums that leave and come back. Us cut / whole, one token through e of 4096 x 7168 (16 e items for 74 pairs):
// e = 5 32 / 37, 6 36 / 38, 7 40 / 39, 8 44 / 42, 9 49 / 45, 10 51 / 56, 12 60 / 58, 14 69 / 74; 256 c rows of 4096 x 4096 (16 c items): c = 5 35 / 32, 8
// 43 / 36, 10 44 / 45, 14 56 / 57, 18 69 / 65, 20 75 / 74; of 4096 x 1024 5 25 / 16, 10 29 / 19, 20 38 / 29.
__host__ __device__ __forceinline__ bool i8_cuts(int over, int pairs, int steps, int chunk) {
    if (over == 0)
        return false;
    const int64_t cost = 4 + chunk / 8, saved = chunk <= 64 ? 55 * int64_t(pairs) - 100 * int64_t(over) : 100 * int64_t(pairs - over);
    return saved * steps > 100 * cost * pairs;
}

// How the items of a launch are dealt out (host-callable, so that a CPU test can walk it): the first `cut` items by ranges of steps,
// pair c's being [cut steps c / ranges, cut steps (c + 1) / ranges); then items cut + c, cut + c + pairs, ...
struct I8Plan {
    int items, cut, ranges, pairs, steps;
    int64_t begin, end;  // this pair's range
    int c;
    __host__ __device__ __forceinline__ I8Plan(int items_, int steps_, int chunk, int pairs_, int c_)
        : items(items_), pairs(pairs_), steps(steps_), c(c_) {
        const int over = items % pairs;
        cut = !i8_cuts(over, pairs, steps, chunk) ? 0 : items < pairs ? items : pairs + over;
        const int64_t total = int64_t(cut) * steps, pieces = total / kI8MinSteps > cut ? total / kI8MinSteps : cut;
        ranges = int(pieces < 1 ? 1 : pieces < pairs ? pieces : pairs);
        begin = c < ranges ? total * c / ranges : 0;
        end = c < ranges ? total * (c + 1) / ranges : 0;
    }
    // The pair whose range holds a step of the cut items.
    __host__ __device__ __forceinline__ int pair_of(int64_t step) const { return int(((step + 1) * ranges - 1) / (int64_t(cut) * steps)); }
    // f(item, first step, steps, first pair of the item, pieces) for each of this pair's pieces, in order.
    template <class F> __host__ __device__ __forceinline__ void pieces(F &&f) const {
        for (int64_t s = begin; s < end;) {
            const int item = int(s / steps);
            const int64_t at = int64_t(item) * steps;
            const int k0 = int(s - at);
            const int n = int(end - s < steps - k0 ? end - s : steps - k0);
            const int first = pair_of(at);
            f(item, k0, n, first, pair_of(at + steps - 1) - first + 1);
            s += n;
        }
        for (int item = cut + c; item < items; item += pairs)
            f(item, 0, steps, c, 1);
    }
};

struct I8Item {
    int e, n0, r0, count, width;  // width: the product's columns, count rounded up to 32
};
// Token chunks of `count` rows, and their size: as equal as steps of 32 allow.
__host__ __device__ __forceinline__ int i8_chunks(int count, int most) { return (count + most - 1) / most; }
__host__ __device__ __forceinline__ int i8_chunk_size(int count, int chunks) { return ((count + chunks - 1) / chunks + 31) & ~31; }
// Where an item lies. A role's items only rise, so the expert and the band of the last one are kept: looked up anew for each item, the
// divisions and the search had cost the products 1100 cycles an item, where one of 2048 k takes 8200.
//   Order of an expert's tiles x chunks: bands of kI8Band tiles, in each the chunks one after the other, each over the band's tiles, so
//   that the pairs at work at one time share a band's weights and a few chunks' tokens in L2.
struct I8Cursor {
    int e = 0, begin = 0, end = 0;      // the expert and its items
    int row = 0, rows = 0, chunks = 0, size = 0;
    int band = 0, band_begin = 0, wide = 0, shift = 0;  // its tiles from kI8Band band on, `wide` of them (2^shift, or shift -1)
    __host__ __device__ __forceinline__ void to_band(int band_, int begin_, int tiles) {
        band = band_;
        band_begin = begin_;
        wide = tiles - band * kI8Band < kI8Band ? tiles - band * kI8Band : kI8Band;
        shift = wide == 8 ? 3 : wide == 4 ? 2 : wide == 2 ? 1 : wide == 1 ? 0 : -1;
    }
    // start: first row of each expert; first: token chunks of the experts before
    __host__ __device__ __forceinline__ I8Item at(int item, int tiles, int experts, const int *start, const int *first) {
        if (item >= end) {
            const int run = item / tiles;
            int lo = e, hi = experts - 1;
            for (int i = 0; i < 4 && lo < hi && first[lo + 1] <= run; ++i)
                ++lo;
            while (lo < hi) {  // the last expert whose first chunk is at or before it
                if (first[lo + 1] > run)
                    break;
                const int mid = (lo + hi + 1) >> 1;
                if (first[mid] <= run)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            e = lo;
            begin = first[e] * tiles;
            end = first[e + 1] * tiles;
            row = start[e];
            rows = start[e + 1] - row;
            chunks = first[e + 1] - first[e];
            size = i8_chunk_size(rows, chunks);
            to_band(0, begin, tiles);
        }
        while (item >= band_begin + wide * chunks)
            to_band(band + 1, band_begin + wide * chunks, tiles);
        const int rest = item - band_begin, chunk = shift >= 0 ? rest >> shift : rest / wide;
        const int left = rows - chunk * size, count = left < size ? left : size;
        return {e, (band * kI8Band + rest - chunk * wide) * kI8TileRows, row + chunk * size, count, (count + 31) & ~31};
    }
};

struct I8Work {
    const int *start, *first;  // shared: first row of each expert (checked), token chunks of the experts before
    int items;
    bool falls;

    // offsets come from the device: each is held to the range that the rows allow, and where they fall no expert gets rows. By all threads
    // of the block, which are together after it. Read from L2, since they are read before the wait where the rows' kernel precedes (I8Params).
    __device__ __forceinline__ I8Work(const I8Params &p, int *start_, int *first_) : start(start_), first(first_) {
        const int E = p.experts, tid = threadIdx.x;
        bool bad = false;
        for (int e = tid; e <= E; e += blockDim.x) {
            const int64_t v = __ldcg(p.offsets + e), before = e ? __ldcg(p.offsets + e - 1) : 0;
            bad |= v < before;
            if (v < before || v > p.rows)
                report(p.status, kSiteOffsets);
            start_[e] = int(max(int64_t(0), min(v, p.rows)));
        }
        falls = __syncthreads_or(bad) != 0;
        auto chunks_of = [&](int e) { return i8_chunks(start[e + 1] - start[e], p.chunk); };
        const int per = (E + int(blockDim.x) - 1) / int(blockDim.x);
        int sum = 0, chunks;
        if (!falls)
            for (int e = tid * per; e < min(E, (tid + 1) * per); ++e)
                sum += chunks_of(e);
        int at = block_scan(sum, chunks);
        if (!falls)
            for (int e = tid * per; e < min(E, (tid + 1) * per); ++e) {
                first_[e] = at;
                at += chunks_of(e);
            }
        if (tid == 0)
            first_[E] = chunks;
        __syncthreads();
        items = chunks * p.tiles;
    }
    __device__ __forceinline__ I8Item at(const I8Params &p, int item, I8Cursor &cursor) const {
        return cursor.at(item, p.tiles, p.experts, start, first);
    }
};

// The rows in expert order: place r gets x[row(r)], rounded to 8 bits where x has 16, and its scale. A block a row (and every gridDim.x-th
// after it). A src that is no slot gives scale 0, so that its row becomes zero.
template <class T> __global__ void __launch_bounds__(512) i8_rows(const __grid_constant__ I8Params p) {
    __shared__ uint32_t part[2][16];
    ptx::griddep_wait();
    // The product kernel may start now: what precedes this one is done (its blocks have waited), and before it reads xq it waits for this one.
    ptx::griddep_launch_dependents();
    const int64_t low = max(0, p.offsets[0]), high = min(p.rows, int64_t(p.offsets[p.experts]));
    if (threadIdx.x == 0 && (p.offsets[0] < 0 || p.offsets[p.experts] > p.rows))
        report(p.status, kSiteOffsets);  // before the src that such offsets reach
    int turn = 0;
    for (int64_t r = low + blockIdx.x; r < high; r += gridDim.x) {
        int64_t row = r;
        if (p.src) {
            const int s = p.src[r];
            row = s < 0 || s >= p.slots ? -1 : s / p.top_k;
        }
        if (row < 0) {
            if (threadIdx.x == 0) {
                report(p.status, kSiteSrc);
                p.xq_scales[r] = 0.0f;
            }
            continue;
        }
        if (p.x_scales) {
            const uint4 *from = reinterpret_cast<const uint4 *>(static_cast<const int8_t *>(p.x) + row * p.k);
            uint4 *to = reinterpret_cast<uint4 *>(p.xq + r * p.k);
            const int pieces = p.k / 16, threads = int(blockDim.x);  // four on their way: a load does not pass the stores before it
#pragma unroll 1
            for (int i = threadIdx.x; i < pieces; i += 4 * threads) {
                uint4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j * threads < pieces)
                        v[j] = from[i + j * threads];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j * threads < pieces)
                        to[i + j * threads] = v[j];
            }
            if (threadIdx.x == 0)
                p.xq_scales[r] = __ldcg(p.x_scales + row);
        } else {
            quant_row<T>(static_cast<const uint8_t *>(p.x) + row * p.k * int64_t(sizeof(T)), p.xq + r * p.k, p.xq_scales + r, p.k / 8, part[turn]);
            turn ^= 1;
        }
    }
}

// The same by tokens, where one goes to several places: each row of x is read and rounded once. i8_places finds each slot's place, inv[src[r]] =
// r, for i8_token_rows. What inv holds from other runs or of slots without a place is known by src, which does not point back; and of places
// that name one slot twice all but one are done by themselves at the end. 16384 tokens of 7168 at 2 places: 150 us by places, 104 by tokens, of which 4 are i8_places.
constexpr int kI8PlaceThreads = 256, kI8TokenPlaces = 32;
__device__ __forceinline__ int2 i8_live(const I8Params &p) {
    return make_int2(max(0, p.offsets[0]), int(min(p.rows, int64_t(p.offsets[p.experts]))));
}
__global__ void __launch_bounds__(kI8PlaceThreads) i8_places(const __grid_constant__ I8Params p) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int2 live = i8_live(p);
    if (threadIdx.x == 0 && (p.offsets[0] < 0 || p.offsets[p.experts] > p.rows))
        report(p.status, kSiteOffsets);  // before the src that such offsets reach
    for (int64_t r = live.x + int64_t(blockIdx.x) * kI8PlaceThreads + threadIdx.x; r < live.y; r += int64_t(gridDim.x) * kI8PlaceThreads) {
        const int s = p.src[r];
        if (s >= 0 && s < p.slots) {
            p.inv[s] = int(r);
        } else {
            report(p.status, kSiteSrc);
            p.xq_scales[r] = 0.0f;
        }
    }
}
template <class T> __global__ void __launch_bounds__(512) i8_token_rows(const __grid_constant__ I8Params p) {
    __shared__ uint32_t part[2][16];
    __shared__ int places[2][kI8TokenPlaces + 1];  // and their number
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();  // as i8_rows
    const int2 live = i8_live(p);
    const int tid = threadIdx.x;
    int turn = 0;
    auto row = [&](int64_t t, auto &&find) {
        int *place = places[turn];
        if (p.x_scales) {
            const uint4 *from = reinterpret_cast<const uint4 *>(static_cast<const int8_t *>(p.x) + t * p.k);
            const int pieces = p.k / 16;
            uint4 v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (tid + i * int(blockDim.x) < pieces)
                    v[i] = from[tid + i * int(blockDim.x)];
            find(place);
            __syncthreads();
            const int n = place[kI8TokenPlaces];
            for (int j = 0; j < n; ++j) {
                uint4 *to = reinterpret_cast<uint4 *>(p.xq + int64_t(place[j]) * p.k);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (tid + i * int(blockDim.x) < pieces)
                        to[tid + i * int(blockDim.x)] = v[i];
                for (int i = tid + 2 * int(blockDim.x); i < pieces; i += blockDim.x)
                    to[i] = from[i];
                if (tid == 0)
                    p.xq_scales[place[j]] = __ldcg(p.x_scales + t);
            }
        } else {
            quant_row<T>(static_cast<const uint8_t *>(p.x) + t * p.k * int64_t(sizeof(T)), p.k / 8, part[turn], [&] { find(place); }, [&](float scale) {
                const int n = place[kI8TokenPlaces];
                if (tid == 0)
                    for (int j = 0; j < n; ++j)
                        p.xq_scales[place[j]] = scale;
                return [&p, place, n](int at, int vecs, uint2 v) {
                    for (int j = 0; j < n; ++j)
                        Vec8<T>::stg_q(p.xq + int64_t(place[j]) * p.k, at, vecs, v);
                };
            });
        }
        turn ^= 1;
    };
    const int64_t tokens = p.slots / p.top_k;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
        row(t, [&](int *place) {
            if (tid >= 32)
                return;
            bool there = false;
            int r = 0;
            if (tid < p.top_k) {
                const int s = int(t) * p.top_k + tid;
                r = p.inv[s];
                there = r >= live.x && r < live.y && p.src[r] == s;
            }
            const unsigned all = __ballot_sync(0xffffffffu, there);
            if (there)
                place[__popc(all & ((1u << tid) - 1u))] = r;
            if (tid == 0)
                place[kI8TokenPlaces] = __popc(all);
        });
    // places whose slot another one has, too
    for (int64_t base = live.x + int64_t(blockIdx.x) * blockDim.x; base < live.y; base += int64_t(gridDim.x) * blockDim.x) {
        const int64_t mine = base + tid;
        bool alone = true;
        if (mine < live.y) {
            const int s = p.src[mine];
            alone = s < 0 || s >= p.slots || p.inv[s] == int(mine);
        }
        if (!__syncthreads_or(!alone))
            continue;
        for (int64_t r = base; r < min(base + blockDim.x, int64_t(live.y)); ++r) {
            const int s = p.src[r];
            if (s < 0 || s >= p.slots || p.inv[s] == int(r))
                continue;
            row(s / p.top_k, [&](int *place) {
                if (tid == 0) {
                    place[0] = int(r);
                    place[kI8TokenPlaces] = 1;
                }
            });
        }
        __syncthreads();
    }
}

// kOnce: weights are read once, as a rule, and leave L2 first.
template <class T, bool kOnce>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_products(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ I8Params p) {
    extern __shared__ __align__(1024) uint8_t i8_smem[];
    __shared__ int start[kI8MaxExperts + 1], first[kI8MaxExperts + 1];
    __shared__ uint64_t bar_mem[2 * kI8MaxStages + 4];
    __shared__ __align__(16) float row_scale[kI8EpilogueWarps][kI8MaxTokens / 2];
    __shared__ uint32_t slots[2];
    const uint32_t ring = (ptx::smem_addr(i8_smem) + 1023u) & ~1023u;
    const uint32_t bars = ptx::smem_addr(bar_mem);
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kI8MaxStages + s); };
    auto tfull = [&](int a) { return bars + 8u * (2 * kI8MaxStages + a); };
    auto tempty = [&](int a) { return bars + 8u * (2 * kI8MaxStages + 2 + a); };
    volatile uint32_t *abort_flag = slots + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            ptx::mbar_init(full(s), p.test_stall && blockIdx.x == 0 && s == 0 ? 2 : 1);
            ptx::mbar_init(empty(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(tfull(a), 1);
            ptx::mbar_init(tempty(a), 2 * kI8EpilogueWarps);  // the epilogue warps of both CTAs
        }
        *abort_flag = 0u;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tmap(&tmap_w);
        ptx::prefetch_tmap(&tmap_x);
    }
    if (warp == 1) {
        ptx::tmem_alloc<2>(ptx::smem_addr(slots), 512);
        ptx::tmem_relinquish<2>();
    }
    ptx::tc_fence_before();
    __syncwarp();
    ptx::cluster_arrive();  // this CTA's barriers are initialised
    if (!p.after_rows)
        ptx::griddep_wait();
    ptx::fence_proxy_async_global();
    ptx::griddep_launch_dependents();
    const I8Work work(p, start, first);
    ptx::cluster_wait();  // and so are the peer's, before any remote arrive
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(slots);
    const Abort ab{p.status + 2, abort_flag, p.timeout_ns};
    const I8Plan plan(work.items, p.steps, p.chunk, pairs, pair);

    if (warp == 0) {
        const uint32_t issue = ptx::elect_one_sync();
        const uint32_t full_leader = ptx::mapa(full(0), 0);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true, waited = !p.after_rows;
        [[maybe_unused]] const uint64_t once = ptx::l2_policy_evict_first();
        I8Cursor cursor;
        plan.pieces([&](int item, int k0, int n, int, int) {
            const I8Item it = work.at(p, item, cursor);
            // A CTA's half of the tokens is one load, of half a chunk's rows whatever the item has (16, 32 or 64 rows a load took 892, 826 and
            // 859 us in place of 700: 8 experts of 4096 rows, 4096 x 7168); where no row of the half is there, none. What is loaded beyond the
            // item's rows, or not at all, goes into sums that nothing reads.
            const int half = it.width / 2, row = it.r0 + int(rank) * half;
            const bool mine = it.count > int(rank) * half;
            const uint32_t bytes = 2u * kI8WeightBytes + (it.count > half ? 2u : 1u) * uint32_t(p.stage_bytes - kI8WeightBytes);
            for (int j = 0; ok && j < n; ++j) {
                ok = wait_all(empty(s), ph ^ 1u, ab, kStatusTimeout | kRoleProducer | uint32_t(s));
                if (!ok)
                    break;
                const uint32_t a = ring + uint32_t(s * p.stage_bytes);
                const int c = (k0 + j) * kI8StepK;
                ptx::mbar_arrive_expect_tx(full(s), bytes, rank == 0 ? issue : 0u);
                if constexpr (kOnce)
                    ptx::tma_load_3d_pair_hint(a, &tmap_w, full_leader + 8u * s, c, it.n0 + int(rank) * 128, it.e, once, issue);
                else
                    ptx::tma_load_3d_pair(a, &tmap_w, full_leader + 8u * s, c, it.n0 + int(rank) * 128, it.e, issue);
                if (!waited) {  // i8_rows' output is read from here on
                    ptx::griddep_wait();
                    ptx::fence_proxy_async_global();
                    waited = true;
                }
                if (mine)
                    ptx::tma_load_2d_pair(a + kI8WeightBytes, &tmap_x, full_leader + 8u * s, c, row, issue);
                if (++s == p.stages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        });
        // every stage released: no commit is still in flight to this CTA
        for (int i = 0; ok && i < p.stages; ++i) {
            ok = wait_all(empty(s), ph ^ 1u, ab, kStatusTimeout | kRoleProducer | 0x80u);
            if (++s == p.stages) {
                s = 0;
                ph ^= 1u;
            }
        }
        if (!waited)
            ptx::griddep_wait();  // this launch ends after i8_rows even where it has no work
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t issue = ptx::elect_one_sync();
            int s = 0;
            uint32_t ph = 0, turn = 0;
            bool ok = true;
            I8Cursor cursor;
            plan.pieces([&](int item, int, int n, int, int) {
                if (!ok)
                    return;
                const I8Item it = work.at(p, item, cursor);
                const uint32_t idesc = i8_idesc(kI8TileRows, it.width);
                const int acc = int(turn & 1u);
                ok = wait_all(tempty(acc), ((turn >> 1) & 1u) ^ 1u, ab, kStatusTimeout | kRoleMma | 0x40u | uint32_t(acc));
                if (!ok)
                    return;
                ptx::tc_fence_after();
                const uint32_t d = tmem + uint32_t(acc * kI8MaxTokens);
                for (int j = 0; j < n; ++j) {
                    ok = wait_all(full(s), ph, ab, kStatusTimeout | kRoleMma | uint32_t(s));
                    if (!ok)
                        return;
                    ptx::tc_fence_after();
                    const uint32_t a = ring + uint32_t(s * p.stage_bytes);
                    const uint64_t ad = ptx::sw128_kmajor_desc(a), bd = ptx::sw128_kmajor_desc(a + kI8WeightBytes);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)  // 32 bytes of k each
                        umma_i8_pair(d, ad + uint64_t(kk * 2), bd + uint64_t(kk * 2), idesc, (j | kk) != 0 ? 1u : 0u, issue);
                    ptx::umma_commit<2>(empty(s), issue);
                    ptx::umma_commit<2>(ptx::mapa(empty(s), 1), issue);
                    if (++s == p.stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                ptx::umma_commit<2>(tfull(acc), issue);
                ptx::umma_commit<2>(ptx::mapa(tfull(acc), 1), issue);
                ++turn;
            });
            // both accumulators released by the epilogue warps of the pair
            for (uint32_t i = turn; ok && i < turn + 2; ++i)
                ok = wait_all(tempty(int(i & 1u)), ((i >> 1) & 1u) ^ 1u, ab, kStatusTimeout | kRoleMma | 0x80u);
        }
    } else {
        const int quarter = warp & 3;  // of Tensor Memory's lanes
        const uint32_t tempty_leader = ptx::mapa(tempty(0), 0);
        T *out = static_cast<T *>(p.out);
        // rows of no expert are zero
        {
            const int64_t low = work.falls ? 0 : start[0], high = work.falls ? 0 : start[p.experts];
            const int64_t pieces = p.n / 8, total = (low + p.rows - high) * pieces;
            for (int64_t i = int64_t(blockIdx.x) * (32 * kI8EpilogueWarps) + (threadIdx.x - 64); i < total; i += int64_t(gridDim.x) * (32 * kI8EpilogueWarps)) {
                const int64_t r = i / pieces, row = r < low ? r : r - low + high;
                reinterpret_cast<uint4 *>(out + row * p.n)[i - r * pieces] = make_uint4(0, 0, 0, 0);
            }
        }
        const int group = (warp - 2) >> 2;  // blocks of 16 tokens that this warp takes: group, group + 2, ...
        float *my_scales = row_scale[warp - 2];
        uint32_t turn = 0;
        bool ok = true;
        I8Cursor cursor;
        plan.pieces([&](int item, int, int, int first_pair, int pieces) {
            if (!ok)
                return;
            const I8Item it = work.at(p, item, cursor);
            const int col = it.n0 + int(rank) * 128 + quarter * 32 + lane, blocks = (it.count + 15) / 16;
            if (p.after_rows && turn == 0)
                ptx::griddep_wait();  // xq_scales are i8_rows' output
            // scales of the rows of this warp's blocks, and of this lane's weight row; whether all are far from the ends of fp32's range
            const float scale = col < p.n ? __ldcg(p.scales + int64_t(it.e) * p.n + col) : 0.0f;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 16 * (group + 4 * i + 2 * (lane >> 4)) + (lane & 15);
                x[i] = j < it.count ? __ldcg(p.xq_scales + it.r0 + j) : 0.0f;
            }
            auto ordinary = [](float v) { return v == 0.0f || (fabsf(v) > 9.0949470e-13f && fabsf(v) < 1.0995116e12f); };  // 2^-40, 2^40
            bool plain = ordinary(scale);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                plain = plain && ordinary(x[i]);
                my_scales[32 * i + lane] = x[i];
            }
            plain = __all_sync(0xffffffffu, plain) != 0;
            const int acc = int(turn & 1u);
            ok = wait_warp(tfull(acc), (turn >> 1) & 1u, ab, kStatusTimeout | kRoleEpilogue | uint32_t(acc));
            if (!ok)
                return;
            ++turn;
            ptx::tc_fence_after();
            const uint32_t from = tmem + (uint32_t(quarter * 32) << 16) + uint32_t(acc * kI8MaxTokens);
            const int64_t most = p.chunk / 16;
            // this quarter's part of pair c's piece: slot 0 where the piece begins inside its item, 1 where it begins it
            auto slot = [&](int c) {
                return reinterpret_cast<int4 *>(p.ws) + (((int64_t(2 * c + (c == first_pair ? 1 : 0)) * 2 + rank) * 4 + quarter) * most) * 128 + lane;
            };
            bool store = true;
            if (pieces > 1 && group < blocks) {
                int32_t *counter = p.counters + (first_pair * 2 + int(rank)) * kI8EpilogueWarps + warp - 2;
                // Where all the others have left theirs, this warp's own sums need not leave Tensor Memory.
                int before = 0;
                if (lane == 0)
                    before = *reinterpret_cast<volatile int32_t *>(counter);
                if (__shfl_sync(0xffffffffu, before, 0) != pieces - 1) {
                    int4 *mine = slot(pair);
#pragma unroll 1
                    for (int b = group; b < blocks; b += 2) {
                        uint32_t r[16];
                        tmem_ld_x16(from + uint32_t(b * 16), r);
                        tmem_wait_ld16(r);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            __stcg(mine + b * 128 + j * 32, make_int4(int(r[4 * j]), int(r[4 * j + 1]), int(r[4 * j + 2]), int(r[4 * j + 3])));
                    }
                    __threadfence();
                    __syncwarp();
                    if (lane == 0)
                        before = atomicAdd(counter, 1);
                    store = __shfl_sync(0xffffffffu, before, 0) == pieces - 1;
                }
                if (store) {
                    __threadfence();
                    if (lane == 0)
                        *counter = 0;  // for the next launch
                }
            }
            if (store) {
                // Two tokens of a lane become two weight rows of one token by an exchange with the lane beside it: even lanes store
                // token j, odd ones j + 1, four bytes each.
                const uint32_t pick = lane & 1 ? 0x3276u : 0x5410u;
                const int64_t row_bytes = int64_t(p.n) * int64_t(sizeof(T));
                uint8_t *to = reinterpret_cast<uint8_t *>(out) + (it.r0 + 16 * group + (lane & 1)) * row_bytes + (col & ~1) * int64_t(sizeof(T));
                int rows = col < p.n ? it.count - 16 * group - (lane & 1) : 0;
                const float *xs = my_scales;
#pragma unroll 1
                for (int b = group; b < blocks; b += 2, to += 32 * row_bytes, rows -= 32, xs += 16) {
                    uint32_t r[16];
                    tmem_ld_x16(from + uint32_t(b * 16), r);
                    tmem_wait_ld16(r);
                    if (pieces > 1)
#pragma unroll 1
                        for (int c = first_pair; c < first_pair + pieces; ++c)
                            if (c != pair) {
                                const int4 *theirs = slot(c) + b * 128;
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const int4 v = __ldcg(theirs + j * 32);
                                    r[4 * j] += uint32_t(v.x);
                                    r[4 * j + 1] += uint32_t(v.y);
                                    r[4 * j + 2] += uint32_t(v.z);
                                    r[4 * j + 3] += uint32_t(v.w);
                                }
                            }
                    // scales near the ends of fp32's range: products that leave it on the way only, in 64 bits
                    if (plain)
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            r[j] = __float_as_uint(float(int(r[j])) * xs[j] * scale);
                    else
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            r[j] = __float_as_uint(float(double(int(r[j])) * double(xs[j]) * double(scale)));
                    uint8_t *at = to;
#pragma unroll
                    for (int j = 0; j < 16; j += 2, at += 2 * row_bytes) {
                        const uint32_t own = moe::pack2<T>(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                        const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
                        if (j < rows)
                            __stcs(reinterpret_cast<uint32_t *>(at), __byte_perm(own, other, pick));
                    }
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive_cluster_cta(tempty_leader + 8u * acc);
        });
    }

    // ---- teardown ----
    __syncwarp();
    if (*abort_flag != 0u) {
        // let copies and MMAs already issued drain before the memory they target goes away
        const uint64_t t0 = ptx::globaltimer();
        while (ptx::globaltimer() - t0 < 200000ull)
            __nanosleep(1000);
        atomicCAS(p.status, 0u, *reinterpret_cast<volatile uint32_t *>(p.status + 2));
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();  // no remote arrive or MMA still targets either CTA
    ptx::tc_fence_after();
    if (warp == 1)
        ptx::tmem_dealloc<2>(tmem, 512);
}

}  // namespace moe
}  // namespace gg
