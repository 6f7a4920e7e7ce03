// Router of a mixture-of-experts layer: top-k experts of each token, their weights, the stable
// order of the (token, choice) slots by expert, per-expert counts and the balance losses; and the
// gradient of weights and losses with respect to the logits.
#pragma once

#include <cmath>

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;
// Warps of a block of route_topk, by logits a lane (V = experts / 32 rounded up to a power of two): as many as the registers
// allow, since a warp waits for its token's row and for its reductions most of the time.
__host__ __device__ constexpr int route_warps(int v) { return v <= 8 ? 32 : v == 16 ? 16 : 8; }
constexpr int kGradWarps = 8;
constexpr int kGradThreads = kGradWarps * 32;
constexpr int kPlaceThreads = 1024;
constexpr int kPlaceCluster = 4;

struct RouteParams {
    const void *logits;   // [tokens, experts]
    const uint8_t *mask;  // [tokens] or null
    int32_t *ids;         // [tokens, top_k]
    float *weights;       // [tokens, top_k]
    float *lse;           // [tokens] or null
    int32_t *counts;      // [experts]
    int32_t *offsets;     // [experts + 1]
    int32_t *live;        // [1]
    int32_t *dest;        // [tokens, top_k]
    int32_t *src;         // [tokens * top_k]
    float *prob;          // [experts] or null
    float *losses;        // [2] or null
    int32_t *block_counts;  // [blocks, experts + 1]: slots of each expert, then live tokens
    float *block_sums;      // [blocks, experts + 1]: probability sums, then the sum of lse^2
    int64_t tokens, per_block;
    int experts, top_k, blocks, normalize;
    int alone;  // one block finishes without route_place: it has a thread an expert
    float scale;
};

struct RouteGradParams {
    const void *logits;
    const uint8_t *mask;
    const int32_t *ids;
    const float *lse;
    const int32_t *counts, *live;
    const float *dweights;  // [tokens, top_k] or null
    const float *dlosses;   // [2] or null
    void *dlogits;
    uint32_t *status;
    int64_t tokens;
    int experts, top_k, normalize;
    float scale;
};

// Logits as unsigned keys in the same order. The addition makes -0 and +0 alike, and every NaN the one NaN that arithmetic gives
// (0x7fffffff), whose key is above +inf's.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;  // key_of(-inf): not to be chosen

// e^x for x <= 0, below 2^-126 as 0: three instructions where results below that cost four more. Relative error (|x| + 4) 2^-24: the
// rounding of the product, as much as the difference behind x had, and ex2.approx's own.
__device__ __forceinline__ float exp_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}

template <class T, int V> __device__ __forceinline__ void load_row(float (&v)[V], const T *row, int experts, bool there) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        v[i] = there && e < experts ? to_f32(row[e]) : -INFINITY;
    }
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// The k largest of a warp's keys (lane + 32 i: expert), ties to the lower expert: lane j < k gets the j-th one's expert and key,
// the others -1. `mine`: the lane's largest key. `list`: 128 words of the warp's.
//
// With L the k-th largest of the lanes' own largest keys, the k largest keys are all at least L, and few others are: those
// candidates, compacted in order of expert, are ranked against one another, a lane each. With 256 experts and k = 8 that is
// about a third of the instructions of k rounds of a maximum over all keys, which remain for more than 32 candidates (ties).
template <int V> __device__ __forceinline__ void top_keys(uint32_t (&key)[V], uint32_t mine, int k, uint32_t *list, int &id, uint32_t &id_key) {
    const int lane = threadIdx.x & 31;
    uint32_t least, m = mine;
    for (int found = 0;;) {
        least = __reduce_max_sync(0xffffffffu, m);
        found += __popc(__ballot_sync(0xffffffffu, m == least));  // all lanes, once none is left
        if (found >= k)
            break;
        m = m == least ? 0u : m;
    }
    least = max(least, kKeyMinusInf + 1);  // fewer lanes than k hold an open expert: every open one is a candidate
    int total = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool in = key[i] >= least;
        const uint32_t all = __ballot_sync(0xffffffffu, in);
        const int at = total + __popc(all & ((1u << lane) - 1u));
        if (in && at < 32)
            reinterpret_cast<uint2 *>(list)[at] = make_uint2(key[i], uint32_t(lane + 32 * i));
        total += __popc(all);
    }
    id = -1;
    id_key = kKeyMinusInf;
    if (total <= 32) {
        __syncwarp();
        const uint2 own = reinterpret_cast<const uint2 *>(list)[lane];
        const uint32_t mykey = lane < total ? own.x : 0u;
        int rank = 0;
        for (int q0 = 0; q0 < total; q0 += 4)  // past the end the keys are 0
#pragma unroll
            for (int q = q0; q < q0 + 4; ++q) {
                const uint32_t other = __shfl_sync(0xffffffffu, mykey, q);
                rank += other > mykey || (other == mykey && q < lane);
            }
        if (lane < total && rank < k)
            reinterpret_cast<uint2 *>(list)[32 + rank] = own;
        __syncwarp();
        if (lane < min(total, k)) {
            const uint2 chosen = reinterpret_cast<const uint2 *>(list)[32 + lane];
            id_key = chosen.x;
            id = int(chosen.y);
        }
        return;
    }
    for (int j = 0; j < k; ++j) {
        uint32_t bk = 0;
        int bi = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (key[i] > bk) {
                bk = key[i];
                bi = lane + 32 * i;
            }
        const uint32_t best = __reduce_max_sync(0xffffffffu, bk);
        if (best <= kKeyMinusInf)
            break;
        const int e = int(__reduce_min_sync(0xffffffffu, bk == best ? unsigned(bi) : 0x7fffffffu));
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (lane + 32 * i == e)
                key[i] = 0;
        if (lane == j) {
            id = e;
            id_key = best;
        }
    }
}

// The totals' outputs and the losses, by one block: tot and sum are the thread's expert's (thread e).
__device__ __forceinline__ void route_totals(const RouteParams &p, int tot, int at, int total, float sum, int live, float z) {
    const int e = threadIdx.x, E = p.experts;
    const float inv = 1.0f / float(max(live, 1));
    float balance = 0.0f;
    if (e < E) {
        p.offsets[e] = at;
        p.counts[e] = tot;
        if (p.prob)
            p.prob[e] = sum * inv;
        balance = float(tot) * (sum * inv);
    }
    if (e == 0) {
        p.offsets[E] = total;
        *p.live = live;
    }
    if (!p.losses)
        return;
    __shared__ float red[32];
    balance = warp_sum(balance);
    if ((e & 31) == 0)
        red[e >> 5] = balance;
    __syncthreads();
    if (e >= 32)
        return;
    const float s = warp_sum(e < int(blockDim.x) >> 5 ? red[e] : 0.0f);
    if (e == 0) {
        p.losses[0] = s * float(E) / float(p.top_k) * inv;
        p.losses[1] = z * inv;
    }
}

// One warp a token, V logits a lane. A block takes a contiguous run of tokens and each of its
// warps a contiguous part of it, so that a warp's own counter of each expert gives the rank of a slot
// among the warp's slots in order; the ranks are raised by the warps before in the block here and by the
// blocks before in route_place, or here where one block takes all tokens. Bound by instruction issue: 710 a token with 256 experts
// and k = 8, 70% of the slots taken. 16384 tokens take 24.1 us with route_place (12% of that for the logits' bytes at the copy rate),
// 1000 tokens of 33 experts 11.2, one token 6.4, which is what the call costs the host.
template <class T, int V> __global__ void __launch_bounds__(route_warps(V) * 32) route_topk(const RouteParams p) {
    constexpr int W = route_warps(V), kThreads = W * 32;
    extern __shared__ int32_t route_smem[];  // [warps][experts] counters, then [warps][128] for top_keys
    __shared__ float z_of[W];
    __shared__ int live_of[W];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int E = p.experts, k = p.top_k;
    const int64_t begin = blockIdx.x * p.per_block, end = min(p.tokens, begin + p.per_block);
    const int64_t per_warp = (p.per_block + W - 1) / W;
    const int64_t w0 = min(end, begin + warp * per_warp), w1 = min(end, w0 + per_warp);
    const int busy = int((end - begin + per_warp - 1) / per_warp);  // warps that have tokens
    int32_t *hist = route_smem + warp * E;
    uint32_t *list = reinterpret_cast<uint32_t *>(route_smem + W * E + warp * 128);
    float v[V];
    auto load = [&](int64_t t) {
        load_row<T, V>(v, static_cast<const T *>(p.logits) + t * E, E, !p.mask || p.mask[t] != 0);
    };
    if (w0 < w1)
        load(w0);
    for (int e = lane; e < E; e += 32)
        hist[e] = 0;
    __syncwarp();
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        acc[i] = 0.0f;
    float z = 0.0f;
    int live = 0;
    for (int64_t t = w0; t < w1; ++t) {
        uint32_t key[V], mine = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            key[i] = key_of(v[i]);
            mine = max(mine, key[i]);
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
        int32_t id = -1;
        float weight = 0.0f, lse = -INFINITY;
        if (top > kKeyMinusInf) {
            const float mx = value_of(top);  // NaN where the row holds one: all that follows is NaN then
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = exp_of(v[i] - mx);
                sum += v[i];
            }
            sum = warp_sum(sum);
            // The logarithm is the accurate one: near lse = 0, of a row with one logit that matters, __logf's absolute error is the whole result's
            // (0.3 us of 24.1 at 16384 tokens of 256 experts). The quotients are approximate, 2 units in the last place: exact ones
            // took 1.1 us more and left weights and prob no nearer to 64 bits (4.5e-7, 1.9e-7), the exponentials' error stands before theirs.
            lse = mx + logf(sum);
            const float inv = __fdividef(1.0f, sum);
#pragma unroll
            for (int i = 0; i < V; ++i)
                acc[i] = fmaf(v[i], inv, acc[i]);
            z = fmaf(lse, lse, z);
            ++live;
            if (t + 1 < w1)
                load(t + 1);  // arrives behind the selection
            uint32_t id_key;
            top_keys<V>(key, mine, k, list, id, id_key);
            const float ex = id >= 0 ? exp_of(value_of(id_key) - mx) : 0.0f;
            weight = p.normalize ? __fdividef(ex, warp_sum(ex)) : ex * inv;
            weight = id >= 0 ? weight * p.scale : 0.0f;
        } else if (t + 1 < w1) {
            load(t + 1);
        }
        if (lane < k) {
            int rank = -1;
            if (id >= 0)
                rank = hist[id]++;  // a token's experts are distinct
            p.ids[t * k + lane] = id;
            p.weights[t * k + lane] = weight;
            p.dest[t * k + lane] = rank;
        }
        if (p.lse && lane == 0)
            p.lse[t] = lse;
        __syncwarp();
    }
    if (lane == 0) {
        z_of[warp] = z;
        live_of[warp] = live;
    }
    __syncthreads();
    const bool alone = p.alone != 0;
    int32_t *counts = p.block_counts + int64_t(blockIdx.x) * (E + 1);
    float *sums = p.block_sums + int64_t(blockIdx.x) * (E + 1);
    int own[(kMaxExperts + kThreads - 1) / kThreads] = {};  // this thread's experts' slots (one expert where a block is alone)
#pragma unroll
    for (int i = 0; i < (kMaxExperts + kThreads - 1) / kThreads; ++i) {
        const int e = tid + i * kThreads;
        if (e >= E)
            break;
        int run = 0;
        for (int w = 0; w < busy; ++w) {
            const int c = route_smem[w * E + e];
            route_smem[w * E + e] = run;
            run += c;
        }
        own[i] = run;
        if (!alone)
            counts[e] = run;
    }
    int n = 0;
    float zs = 0.0f;
    for (int w = 0; w < busy; ++w) {
        n += live_of[w];
        zs += z_of[w];
    }
    if (!alone && tid == 0) {
        counts[E] = n;
        sums[E] = zs;
    }
    int at = 0, total = 0;
    if (alone) {  // route_place's part too: the experts' first places into the warps' counters
        at = block_scan(own[0], total);
        if (tid < E)
            for (int w = 0; w < busy; ++w)
                route_smem[w * E + tid] += at;
    }
    __syncthreads();
    for (int64_t s = w0 * k + lane; s < w1 * k; s += 32) {
        const int id = p.ids[s];
        if (id >= 0) {
            const int d = p.dest[s] + hist[id];
            p.dest[s] = d;
            if (alone)
                p.src[d] = int(s);
        }
    }
    if (alone)
        for (int64_t r = total + tid; r < p.tokens * k; r += kThreads)
            p.src[r] = -1;
    if (!p.prob && !p.losses) {
        if (alone)
            route_totals(p, own[0], at, total, 0.0f, n, zs);
        return;
    }
    __syncthreads();
    float *part = reinterpret_cast<float *>(route_smem);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (lane + 32 * i < E)
            part[warp * E + lane + 32 * i] = acc[i];
    __syncthreads();
    float mine = 0.0f;
    for (int e = tid; e < E; e += kThreads) {
        float s = 0.0f;
        for (int w = 0; w < busy; ++w)
            s += part[w * E + e];
        if (!alone)
            sums[e] = s;
        mine = s;
    }
    if (alone)
        route_totals(p, own[0], at, total, mine, n, zs);
}

// Every block needs the blocks' counts (all of them for the experts' offsets, those before it for its own
// slots); it places its slots and writes its part of src's unused end; one block more writes the totals and losses. Its 1024
// threads share the blocks' rows of an expert: 37 loads a thread for 148 rows of 256 experts. Where that is much, a cluster of C
// blocks shares the sums: each adds every C-th row and reads the others' sums from their shared memory, and adds the few rows of
// its own cluster before it.
template <int C> __global__ void __launch_bounds__(kPlaceThreads) route_place(const RouteParams p) {
    __shared__ int part[2][kPlaceThreads];
    __shared__ int base[kMaxExperts];
    __shared__ int share[C > 1 ? 3 : 1][C > 1 ? kPlaceThreads : 1];  // this block's part of tot, pre and sum
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int E = p.experts, k = p.top_k, tid = threadIdx.x, b = blockIdx.x;
    const int turn = b % C, c0 = b - turn;  // c0: the cluster's first block
    const bool last = b == p.blocks, sums = p.blocks - c0 < C && (p.prob || p.losses);
    const int mine = (p.blocks - turn + C - 1) / C;  // rows of this block's part: turn, turn + C, ...
    int span = 32;  // a power of two of at least E threads takes one row
    while (span < E)
        span *= 2;
    const int rows = kPlaceThreads / span, e = tid % span, row = tid / span;
    // the thread's first slot, on its way while the counts are summed
    const int64_t first = min(p.tokens, b * p.per_block) * k, end = min(p.tokens, (b + 1) * p.per_block) * k;
    int id0 = -1, rank0 = 0;
    if (first + tid < end) {
        id0 = p.ids[first + tid];
        rank0 = p.dest[first + tid];
    }
    int tot = 0, pre = 0;
    float sum = 0.0f;
    if (e < E) {
        for (int r0 = row; r0 < mine; r0 += 8 * rows) {  // eight rows' loads at a time (16 and more at once were slower)
            int c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                c[i] = r0 + i * rows < mine ? __ldcg(p.block_counts + (turn + C * (r0 + i * rows)) * (E + 1) + e) : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                tot += c[i];
                pre += turn + C * (r0 + i * rows) < c0 ? c[i] : 0;
            }
        }
        if (sums)
            for (int r0 = row; r0 < mine; r0 += 8 * rows) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    f[i] = r0 + i * rows < mine ? __ldcg(p.block_sums + (turn + C * (r0 + i * rows)) * (E + 1) + e) : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sum += f[i];
            }
    }
    int near = 0;
    if (tid < E)
        for (int i = c0; i < min(b, p.blocks); ++i)
            near += __ldcg(p.block_counts + i * (E + 1) + tid);
    auto across = [&](auto v, auto *words) {  // of the threads of one expert, in order; complete in the first
        words[tid] = v;
        __syncthreads();
        if (tid < span)
            for (int r = 1; r < rows; ++r)
                v += words[r * span + tid];
        __syncthreads();
        return v;
    };
    tot = across(tot, part[0]);
    pre = across(pre, part[1]);
    if (sums)
        sum = across(sum, reinterpret_cast<float *>(part[0]));
    if constexpr (C > 1) {
        share[0][tid] = tot;
        share[1][tid] = pre;
        share[2][tid] = __float_as_int(sum);
        ptx::cluster_sync();
        tot = pre = 0;
        sum = 0.0f;
        if (tid < E)
#pragma unroll
            for (int q = 0; q < C; ++q) {
                tot += int(ld_cluster_u32(ptx::mapa(ptx::smem_addr(&share[0][tid]), q)));
                pre += int(ld_cluster_u32(ptx::mapa(ptx::smem_addr(&share[1][tid]), q)));
                if (sums)
                    sum += __uint_as_float(ld_cluster_u32(ptx::mapa(ptx::smem_addr(&share[2][tid]), q)));
            }
        ptx::cluster_sync();  // no block ends while another still reads from it
    }
    if (b > p.blocks)
        return;
    pre += near;
    if (tid >= E)
        tot = 0;
    int total;
    const int at = block_scan(tot, total);
    if (last) {
        int live = 0;
        float z = 0.0f;
        for (int r = tid; r < p.blocks; r += kPlaceThreads) {  // blocks: at most one a thread
            live += p.block_counts[int64_t(r) * (E + 1) + E];
            z += p.block_sums[int64_t(r) * (E + 1) + E];
        }
        part[0][tid] = live;
        part[1][tid] = __float_as_int(z);
        __syncthreads();
        live = 0;
        z = 0.0f;
        if (tid < 32) {
            for (int r = tid; r < kPlaceThreads; r += 32) {
                live += part[0][r];
                z += __int_as_float(part[1][r]);
            }
            live = __reduce_add_sync(0xffffffffu, live);
            z = warp_sum(z);
            part[0][0] = live;
        }
        __syncthreads();
        route_totals(p, tot, at, total, sum, part[0][0], z);
        return;
    }
    if (tid < E)
        base[tid] = at + pre;
    __syncthreads();
    for (int64_t s = first + tid; s < end; s += kPlaceThreads) {
        const bool head = s == first + tid;
        const int id = head ? id0 : p.ids[s];
        if (id >= 0) {
            const int d = (head ? rank0 : p.dest[s]) + base[id];
            p.dest[s] = d;
            p.src[d] = int(s);
        }
    }
    for (int64_t r = total + int64_t(b) * kPlaceThreads + tid; r < p.tokens * k; r += int64_t(p.blocks) * kPlaceThreads)
        p.src[r] = -1;
}

// One warp a token:  d l_e = p_e (g_e - sum p g - sum_j [plain weights] p_j s dw_j + 2 dz lse / live) + add_e
// with p = exp(l - lse), g_e = dbal E c_e / (k live^2), and add the slots' own part:
// p_j s dw_j for plain weights, q_j s (dw_j - sum q dw) for normalised ones (q: softmax over the chosen). The balance term's g is
// the same for all tokens and stays in registers, the slots' part meets the row in shared memory. A row is loaded while the one
// before is computed. 16384 tokens of 256 experts take 12.6 us, 42% of the copy rate for logits in and gradient out: a row's reductions
// and the few rows in flight (24 warps an SM; more warps with fewer registers were slower) bind it.
template <class T, int V> __global__ void __launch_bounds__(kGradThreads) route_grad(const RouteGradParams p) {
    extern __shared__ float grad_smem[];  // per warp the slots' part [experts], zero between tokens
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int E = p.experts, k = p.top_k;
    float *add = grad_smem + E * warp;
    const float n = float(max(*p.live, 1));
    const float db = p.dlosses ? p.dlosses[0] * float(E) / (float(k) * n * n) : 0.0f;
    const float dz = p.dlosses ? 2.0f * p.dlosses[1] / n : 0.0f;
    float bal[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        bal[i] = e < E ? db * float(p.counts[e]) : 0.0f;
        if (e < E)
            add[e] = 0.0f;
    }
    __syncwarp();
    struct Row {
        float v[V], lse, dw;
        int id;
    } next;
    // what a token's gradient needs: its row, lse, and in lane j slot j's expert and scaled gradient
    auto load = [&](int64_t t) {
        const float lse = p.lse[t];
        next.lse = p.mask && p.mask[t] == 0 ? -INFINITY : lse;
        load_row<T, V>(next.v, static_cast<const T *>(p.logits) + t * E, E, true);
        next.id = -1;
        next.dw = 0.0f;
        if (p.dweights && lane < k) {
            next.id = p.ids[t * k + lane];
            next.dw = p.dweights[t * k + lane] * p.scale;
        }
    };
    const int64_t stride = int64_t(gridDim.x) * kGradWarps;
    int64_t t = int64_t(blockIdx.x) * kGradWarps + warp;
    if (t < p.tokens)
        load(t);
    for (; t < p.tokens; t += stride) {
        Row r = next;
        if (t + stride < p.tokens)
            load(t + stride);
        T *out = static_cast<T *>(p.dlogits) + t * E;
        if (r.lse == -INFINITY) {  // not live
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (lane + 32 * i < E)
                    out[lane + 32 * i] = from_f32<T>(0.0f);
            continue;
        }
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            r.v[i] = exp_of(r.v[i] - r.lse);
            dot = fmaf(r.v[i], bal[i], dot);
        }
        if (p.dweights) {
            if (r.id < -1 || r.id >= E) {
                report(p.status, kSiteExpert);
                r.id = -1;
            }
            const bool slot = r.id >= 0;
            const float l = slot ? to_f32(static_cast<const T *>(p.logits)[t * E + r.id]) : -INFINITY;
            const float dw = slot ? r.dw : 0.0f;
            float mine;
            if (p.normalize) {
                float mx = l;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float ex = slot ? exp_of(l - mx) : 0.0f;
                const float sum = warp_sum(ex);
                const float q = slot ? ex / sum : 0.0f;
                mine = q * (dw - warp_sum(q * dw));
            } else {
                mine = slot ? exp_of(l - r.lse) * dw : 0.0f;
                dot += mine;
            }
            if (slot)
                atomicAdd(&add[r.id], mine);  // one addend a place: a token's experts are distinct
        }
        dot = warp_sum(dot);
        __syncwarp();
        const float c = dz * r.lse - dot;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = lane + 32 * i;
            if (e < E)
                out[e] = from_f32<T>(fmaf(r.v[i], bal[i] + c, add[e]));
        }
        __syncwarp();
        if (r.id >= 0)
            add[r.id] = 0.0f;
        __syncwarp();
    }
}

}  // namespace moe
}  // namespace gg
