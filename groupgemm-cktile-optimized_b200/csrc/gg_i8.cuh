// Rows in expert order times their expert's 8-bit weights, with a scale a row and a scale a weight row:
//   out[r, n] = x_scales[row(r)] * scales[e, n] * sum_k x[row(r), k] w[e, n, k]
//
// The sums are whole numbers, exact in 32 bits (k <= kI8MaxK), so neither how the work is cut nor who adds up changes a result.
//
// tcgen05.mma kind::i8 on CTA pairs, the weights as A (256 rows a pair) and a chunk of tokens as B, as wide as the chunk has tokens
// (32 to 256 in steps of 32): few rows an expert cost the bytes of its weights and next to no products, many rows run at the full
// tile, and nothing is padded to a tile of tokens. Tokens are fetched through src by TMA gathers of four rows, so no copy in expert order is made.
//
//   Work split: items (expert, token chunk, 256 weight rows). Each pair takes whole items in turn; the items that would leave pairs
//   idle at the end (or all, where there are few) are cut along k into equal ranges of steps, one a pair, taken first. What is cut
//   leaves its sums in the workspace, and the last warp to arrive adds them up (no order to keep).
//   Warps: 0 loads (weights and tokens, a ring of stages), 1 issues the products (of the pair's first CTA), 2-5 take the sums out of
//   Tensor Memory, two accumulators in turn.
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
constexpr int kI8Threads = 192;
constexpr int kI8Smem = kI8Ring + 1024;
constexpr int kI8Band = 8;          // tiles whose weights are visited together (see item)
constexpr int kI8MinSteps = 4;      // of a cut piece

struct I8Params {
    QuantParams quant;        // first: the parameters of quant_rows, where the rows come in 16 bits
    const float *x_scales;    // [tokens or rows]
    const float *scales;      // [experts, n]
    const int32_t *offsets;   // [experts + 1]
    const int32_t *src;       // [rows] slots, or null: row r is x[r]
    void *out;                // [rows, n]
    uint32_t *status;         // [0] status word, [2] timeouts of this launch
    int32_t *ws;              // [2 x pairs][2 CTAs][4 warps][chunk / 32][8][32] int4
    int32_t *counters;        // [pairs][2][4], 0 between launches
    int64_t rows, slots;      // slots: tokens * top_k
    uint64_t timeout_ns;
    int n, k, experts, top_k, tiles, steps;
    int chunk;                // most tokens of a chunk, a multiple of 32
    int stages, stage_bytes;
    int after_quant;          // 1: quant_rows precedes, and everything before it is done when this kernel starts
};

// Four rows of a 2-D map into one 512-byte piece; the completion barrier may be the pair leader's.
__device__ __forceinline__ void tma_gather4_pair(uint32_t dst, const void *tmap, uint32_t bar, int32_t c, int4 rows, uint32_t pred) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %8, 0;\n\t"
                 "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2"
                 " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n\t}" ::"r"(dst),
                 "l"(tmap), "r"(bar), "r"(c), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(pred)
                 : "memory");
}

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

// How the items of a launch are dealt out (host-callable, so that a CPU test can walk it): the first `cut` items by ranges of steps,
// pair c's being [cut steps c / ranges, cut steps (c + 1) / ranges); then items cut + c, cut + c + pairs, ...
struct I8Plan {
    int64_t items;
    int cut, ranges, pairs, steps;
    int64_t begin, end;  // this pair's range
    int c;
    __host__ __device__ __forceinline__ I8Plan(int64_t items_, int steps_, int pairs_, int c_) : items(items_), pairs(pairs_), steps(steps_), c(c_) {
        const int64_t over = items % pairs;
        cut = over == 0 ? 0 : int(items < pairs ? items : pairs + over);
        const int64_t total = int64_t(cut) * steps, most = total / kI8MinSteps;
        ranges = int(most < 1 ? 1 : most < pairs ? most : pairs);
        begin = c < ranges ? total * c / ranges : 0;
        end = c < ranges ? total * (c + 1) / ranges : 0;
    }
    // The pair whose range holds a step of the cut items.
    __host__ __device__ __forceinline__ int pair_of(int64_t step) const { return int(((step + 1) * ranges - 1) / (int64_t(cut) * steps)); }
    // f(item, first step, steps, first pair of the item, pieces) for each of this pair's pieces, in order.
    template <class F> __host__ __device__ __forceinline__ void pieces(F &&f) const {
        for (int64_t s = begin; s < end;) {
            const int64_t item = s / steps;
            const int k0 = int(s - item * steps);
            const int n = int(end - s < steps - k0 ? end - s : steps - k0);
            const int first = pair_of(item * steps);
            f(item, k0, n, first, pair_of(item * steps + steps - 1) - first + 1);
            s += n;
        }
        for (int64_t item = cut + c; item < items; item += pairs)
            f(item, 0, steps, c, 1);
    }
};

struct I8Item {
    int e, n0, r0, count, width;  // width: the product's columns, count rounded up to 32
};
// Token chunks of `count` rows, and their size: as equal as steps of 32 allow.
__host__ __device__ __forceinline__ int i8_chunks(int count, int most) { return (count + most - 1) / most; }
__host__ __device__ __forceinline__ int i8_chunk_size(int count, int chunks) { return ((count + chunks - 1) / chunks + 31) & ~31; }
// Item `in` of an expert's tiles x chunks: bands of kI8Band tiles, in each the chunks one after the other, each over the band's tiles, so that
// the pairs at work at one time share a band's weights and a few chunks' tokens in L2.
__host__ __device__ __forceinline__ void i8_place(int in, int tiles, int chunks, int &tile, int &chunk) {
    const int band = in / (kI8Band * chunks), rest = in - band * (kI8Band * chunks);
    const int wide = tiles - band * kI8Band < kI8Band ? tiles - band * kI8Band : kI8Band;
    chunk = rest / wide;
    tile = band * kI8Band + rest - chunk * wide;
}

struct I8Work {
    const int *start, *first;  // shared: first row of each expert (checked), token chunks of the experts before
    int64_t items;
    bool falls;

    // offsets come from the device: each is held to the range that the rows allow, and where they fall no expert gets rows. By all threads
    // of the block, which are together after it.
    __device__ __forceinline__ I8Work(const I8Params &p, int *start_, int *first_) : start(start_), first(first_) {
        const int E = p.experts, tid = threadIdx.x;
        bool bad = false;
        for (int e = tid; e <= E; e += blockDim.x) {
            const int64_t v = p.offsets[e], before = e ? p.offsets[e - 1] : 0;
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
        items = int64_t(chunks) * p.tiles;
    }
    __device__ __forceinline__ I8Item at(const I8Params &p, int64_t item) const {
        const int run = int(item / p.tiles);
        int lo = 0, hi = p.experts - 1;  // the last expert whose first chunk is at or before it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= run)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int chunks = first[lo + 1] - first[lo], rows = start[lo + 1] - start[lo], size = i8_chunk_size(rows, chunks);
        int tile, chunk;
        i8_place(int(item - int64_t(first[lo]) * p.tiles), p.tiles, chunks, tile, chunk);
        const int count = min(size, rows - chunk * size);
        return {lo, tile * kI8TileRows, start[lo] + chunk * size, count, (count + 31) & ~31};
    }
};

// The row of x behind place r of the expert order, or -1 (and a report) where src holds no slot.
__device__ __forceinline__ int i8_row(const I8Params &p, int r, bool tell) {
    if (!p.src)
        return r;
    const int s = __ldg(p.src + r);
    if (s >= 0 && s < p.slots)
        return s / p.top_k;
    if (tell)
        report(p.status, kSiteSrc);
    return -1;
}

template <class T>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_products(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ I8Params p) {
    extern __shared__ __align__(1024) uint8_t i8_smem[];
    __shared__ int start[kI8MaxExperts + 1], first[kI8MaxExperts + 1];
    __shared__ uint64_t bar_mem[2 * kI8MaxStages + 4];
    __shared__ float row_scale[4][kI8MaxTokens];
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
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(tfull(a), 1);
            ptx::mbar_init(tempty(a), 8);  // the epilogue warps of both CTAs
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
    if (!p.after_quant)
        ptx::griddep_wait();
    ptx::fence_proxy_async_global();
    ptx::griddep_launch_dependents();
    const I8Work work(p, start, first);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();  // the peer's barriers are initialised before any remote arrive
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(slots);
    const Abort ab{p.status + 2, abort_flag, p.timeout_ns};
    const I8Plan plan(work.items, p.steps, pairs, pair);

    if (warp == 0) {
        const uint32_t issue = ptx::elect_one_sync();
        const uint32_t full_leader = ptx::mapa(full(0), 0);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true, waited = !p.after_quant;
        plan.pieces([&](int64_t item, int k0, int n, int, int) {
            const I8Item it = work.at(p, item);
            const int half = it.width / 2;  // tokens of this CTA
            // lane l gathers tokens 4 l to 4 l + 3 of them; a missing one is read as row 0, its sums go nowhere
            int row[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = int(rank) * half + 4 * lane + i;
                row[i] = 4 * lane < half && j < it.count ? max(0, i8_row(p, it.r0 + j, it.n0 == 0 && k0 == 0)) : 0;
            }
            const int4 rows = make_int4(row[0], row[1], row[2], row[3]);
            const uint32_t gathers = 4 * lane < half ? 1u : 0u;
            for (int j = 0; ok && j < n; ++j) {
                ok = wait_all(empty(s), ph ^ 1u, ab, kStatusTimeout | kRoleProducer | uint32_t(s));
                if (!ok)
                    break;
                const uint32_t a = ring + uint32_t(s * p.stage_bytes);
                const int c = (k0 + j) * kI8StepK;
                ptx::mbar_arrive_expect_tx(full(s), 2u * (kI8WeightBytes + uint32_t(half) * kI8StepK), rank == 0 ? issue : 0u);
                ptx::tma_load_3d_pair(a, &tmap_w, full_leader + 8u * s, c, it.n0 + int(rank) * 128, it.e, issue);
                if (!waited) {  // quant_rows' output is read from here on
                    ptx::griddep_wait();
                    ptx::fence_proxy_async_global();
                    waited = true;
                }
                tma_gather4_pair(a + kI8WeightBytes + uint32_t(lane) * 512u, &tmap_x, full_leader + 8u * s, c, rows, gathers);
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
            ptx::griddep_wait();  // this launch ends after quant_rows even where it has no work
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t issue = ptx::elect_one_sync();
            int s = 0;
            uint32_t ph = 0, turn = 0;
            bool ok = true;
            plan.pieces([&](int64_t item, int, int n, int, int) {
                if (!ok)
                    return;
                const I8Item it = work.at(p, item);
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
            for (int64_t i = int64_t(blockIdx.x) * 128 + (threadIdx.x - 64); i < total; i += int64_t(gridDim.x) * 128) {
                const int64_t r = i / pieces, row = r < low ? r : r - low + high;
                reinterpret_cast<uint4 *>(out + row * p.n)[i - r * pieces] = make_uint4(0, 0, 0, 0);
            }
        }
        uint32_t turn = 0;
        bool ok = true;
        plan.pieces([&](int64_t item, int, int, int first_pair, int pieces) {
            if (!ok)
                return;
            const I8Item it = work.at(p, item);
            const int col = it.n0 + int(rank) * 128 + quarter * 32 + lane;
            if (p.after_quant && turn == 0)
                ptx::griddep_wait();  // x_scales are quant_rows' output
            // scales of the chunk's rows, each warp its own copy
            __syncwarp();
            for (int j = lane; j < it.width; j += 32) {
                const int row = j < it.count ? i8_row(p, it.r0 + j, false) : -1;
                row_scale[quarter][j] = row < 0 ? 0.0f : __ldg(p.x_scales + row);
            }
            const float scale = col < p.n ? __ldg(p.scales + int64_t(it.e) * p.n + col) : 0.0f;
            __syncwarp();
            const int acc = int(turn & 1u);
            ok = wait_warp(tfull(acc), (turn >> 1) & 1u, ab, kStatusTimeout | kRoleEpilogue | uint32_t(acc));
            if (!ok)
                return;
            ++turn;
            ptx::tc_fence_after();
            const uint32_t from = tmem + (uint32_t(quarter * 32) << 16) + uint32_t(acc * kI8MaxTokens);
            const int blocks = it.width / 32;
            const int64_t most = p.chunk / 32;
            // this warp's part of pair c's piece: slot 0 where the piece begins inside its item, 1 where it begins it
            auto slot = [&](int c) {
                return reinterpret_cast<int4 *>(p.ws) + (((int64_t(2 * c + (c == first_pair ? 1 : 0)) * 2 + rank) * 4 + quarter) * most) * 256 + lane;
            };
            bool store = true;
            if (pieces > 1) {
                int32_t *counter = p.counters + (first_pair * 2 + int(rank)) * 4 + quarter;
                int4 *mine = slot(pair);
#pragma unroll 1
                for (int b = 0; b < blocks; ++b) {
                    uint32_t r[32];
                    ptx::tmem_ld_32x32b_x32(from + uint32_t(b * 32), r);
                    ptx::tmem_wait_ld(r);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        __stcg(mine + b * 256 + j * 32, make_int4(int(r[4 * j]), int(r[4 * j + 1]), int(r[4 * j + 2]), int(r[4 * j + 3])));
                }
                __threadfence();
                __syncwarp();
                int before = 0;
                if (lane == 0)
                    before = atomicAdd(counter, 1);
                store = __shfl_sync(0xffffffffu, before, 0) == pieces - 1;
                if (store) {
                    __threadfence();
                    if (lane == 0)
                        *counter = 0;  // for the next launch
                }
            }
            if (store) {
#pragma unroll 1
                for (int b = 0; b < blocks; ++b) {
                    uint32_t r[32];
                    ptx::tmem_ld_32x32b_x32(from + uint32_t(b * 32), r);
                    ptx::tmem_wait_ld(r);
                    for (int c = first_pair; c < first_pair + pieces; ++c)
                        if (c != pair) {
                            const int4 *theirs = slot(c) + b * 256;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int4 v = __ldcg(theirs + j * 32);
                                r[4 * j] += uint32_t(v.x);
                                r[4 * j + 1] += uint32_t(v.y);
                                r[4 * j + 2] += uint32_t(v.z);
                                r[4 * j + 3] += uint32_t(v.w);
                            }
                        }
                    if (col < p.n) {
                        T *to = out + int64_t(it.r0 + b * 32) * p.n + col;
                        const int rows = it.count - b * 32;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j < rows) {
                                // the smaller scale first: no product on the way leaves fp32's range unless the result does
                                const float x = row_scale[quarter][b * 32 + j];
                                const bool less = fabsf(x) < fabsf(scale);
                                const float v = float(int(r[j])) * (less ? x : scale) * (less ? scale : x);
                                to[int64_t(j) * p.n] = from_f32<T>(v);
                            }
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
