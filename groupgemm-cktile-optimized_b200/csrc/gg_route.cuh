// Router of a mixture-of-experts layer: top-k experts of each token, their weights, the stable
// order of the (token, choice) slots by expert, per-expert counts and the balance losses; and the
// gradient of weights and losses with respect to the logits.
#pragma once

#include <cmath>

#include "gg_moe.cuh"

namespace gg {
namespace moe {

constexpr int kRouteWarps = 8;
constexpr int kRouteThreads = kRouteWarps * 32;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;

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

// Logits as unsigned keys in the same order: -0 and +0 alike, every NaN alike and above +inf.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v)
        return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;  // key_of(-inf): not to be chosen

template <class T, int V> __device__ __forceinline__ void load_row(float (&v)[V], const T *row, int experts, bool there) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        v[i] = there && e < experts ? to_f32(row[e]) : -INFINITY;
    }
}

// One warp a token, V logits a lane. A block takes a contiguous run of tokens and each of its
// warps a contiguous part of it, so that a warp's own counter of each expert gives the rank of a slot
// among the warp's slots in order; the ranks are raised by the warps before in the block here and by the
// blocks before in route_place.
template <class T, int V> __global__ void __launch_bounds__(kRouteThreads) route_topk(const RouteParams p) {
    extern __shared__ int32_t route_smem[];  // [warps][experts]
    __shared__ float z_of[kRouteWarps];
    __shared__ int live_of[kRouteWarps];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int E = p.experts, k = p.top_k;
    const int64_t first = blockIdx.x * p.per_block, end = min(p.tokens, first + p.per_block);
    const int64_t per_warp = (p.per_block + kRouteWarps - 1) / kRouteWarps;
    const int64_t w0 = min(end, first + warp * per_warp), w1 = min(end, w0 + per_warp);
    int32_t *hist = route_smem + warp * E;
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
        const bool there = !p.mask || p.mask[t] != 0;
        float v[V];
        load_row<T, V>(v, static_cast<const T *>(p.logits) + t * E, E, there);
        uint32_t key[V], best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            key[i] = key_of(v[i]);
            best = max(best, key[i]);
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        int32_t id = -1;
        float weight = 0.0f, lse = -INFINITY;
        if (top > kKeyMinusInf) {
            const float mx = value_of(top);  // NaN where the row holds one: all that follows is NaN then
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = expf(v[i] - mx);
                sum += v[i];
            }
            sum = warp_sum(sum);
            lse = mx + logf(sum);
            const float inv = 1.0f / sum;
#pragma unroll
            for (int i = 0; i < V; ++i)
                acc[i] += v[i] * inv;
            z += lse * lse;
            ++live;
            uint32_t mine = kKeyMinusInf;
            for (int j = 0; j < k; ++j) {
                uint32_t bk = 0;
                int bi = 0;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (key[i] > bk) {
                        bk = key[i];
                        bi = lane + 32 * i;
                    }
                const uint32_t m = __reduce_max_sync(0xffffffffu, bk);
                if (m <= kKeyMinusInf)
                    break;
                const int e = int(__reduce_min_sync(0xffffffffu, bk == m ? unsigned(bi) : 0x7fffffffu));
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (lane + 32 * i == e)
                        key[i] = 0;
                if (lane == j) {
                    id = e;
                    mine = m;
                }
            }
            const float ex = id >= 0 ? expf(value_of(mine) - mx) : 0.0f;
            weight = p.normalize ? ex / warp_sum(ex) : ex * inv;
            weight = id >= 0 ? weight * p.scale : 0.0f;
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
    int32_t *counts = p.block_counts + int64_t(blockIdx.x) * (E + 1);
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        int run = 0;
        for (int w = 0; w < kRouteWarps; ++w) {
            const int c = route_smem[w * E + e];
            route_smem[w * E + e] = run;
            run += c;
        }
        counts[e] = run;
    }
    if (threadIdx.x == 0) {
        int n = 0;
        float s = 0.0f;
        for (int w = 0; w < kRouteWarps; ++w) {
            n += live_of[w];
            s += z_of[w];
        }
        counts[E] = n;
        p.block_sums[int64_t(blockIdx.x) * (E + 1) + E] = s;
    }
    __syncthreads();
    for (int64_t s = w0 * k + lane; s < w1 * k; s += 32) {
        const int id = p.ids[s];
        if (id >= 0)
            p.dest[s] += hist[id];
    }
    __syncthreads();
    float *sums = reinterpret_cast<float *>(route_smem);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (lane + 32 * i < E)
            sums[warp * E + lane + 32 * i] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        float s = 0.0f;
        for (int w = 0; w < kRouteWarps; ++w)
            s += sums[w * E + e];
        p.block_sums[int64_t(blockIdx.x) * (E + 1) + e] = s;
    }
}

// Every block sums the blocks' counts (all of them for the experts' offsets, those before it for its own
// slots), places its slots and writes its part of src's unused end; block 0 writes the totals.
__global__ void __launch_bounds__(kRouteThreads) route_place(const RouteParams p) {
    __shared__ int base[kMaxExperts];
    __shared__ float red[kRouteWarps];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int E = p.experts, k = p.top_k, tid = threadIdx.x;
    constexpr int kPer = kMaxExperts / kRouteThreads;
    int tot[kPer], pre[kPer], sum = 0;
    const int per = (E + kRouteThreads - 1) / kRouteThreads;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        tot[i] = pre[i] = 0;
        const int e = tid * per + i;
        if (i < per && e < E)
            for (int b = 0; b < p.blocks; ++b) {
                const int c = p.block_counts[int64_t(b) * (E + 1) + e];
                tot[i] += c;
                if (b < int(blockIdx.x))
                    pre[i] += c;
            }
        sum += tot[i];
    }
    int total;
    int at = block_scan(sum, total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * per + i;
        if (i < per && e < E) {
            base[e] = at + pre[i];
            if (blockIdx.x == 0) {
                p.offsets[e] = at;
                p.counts[e] = tot[i];
            }
        }
        at += tot[i];
    }
    __syncthreads();
    const int64_t first = min(p.tokens, blockIdx.x * p.per_block) * k, end = min(p.tokens, (blockIdx.x + 1) * p.per_block) * k;
    for (int64_t s = first + tid; s < end; s += kRouteThreads) {
        const int id = p.ids[s];
        if (id >= 0) {
            const int d = p.dest[s] + base[id];
            p.dest[s] = d;
            p.src[d] = int(s);
        }
    }
    for (int64_t r = total + int64_t(blockIdx.x) * kRouteThreads + tid; r < p.tokens * k; r += int64_t(p.blocks) * kRouteThreads)
        p.src[r] = -1;
    if (blockIdx.x != 0)
        return;
    int live = 0;
    float z = 0.0f;
    for (int b = 0; b < p.blocks; ++b) {
        live += p.block_counts[int64_t(b) * (E + 1) + E];
        z += p.block_sums[int64_t(b) * (E + 1) + E];
    }
    if (tid == 0) {
        p.offsets[E] = total;
        *p.live = live;
    }
    if (!p.prob && !p.losses)
        return;
    const float inv = 1.0f / float(max(live, 1));
    float balance = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * per + i;
        if (i < per && e < E) {
            float s = 0.0f;
            for (int b = 0; b < p.blocks; ++b)
                s += p.block_sums[int64_t(b) * (E + 1) + e];
            s *= inv;
            if (p.prob)
                p.prob[e] = s;
            balance += float(tot[i]) * s;
        }
    }
    balance = warp_sum(balance);
    if ((tid & 31) == 0)
        red[tid >> 5] = balance;
    __syncthreads();
    if (tid == 0 && p.losses) {
        float s = 0.0f;
        for (int w = 0; w < kRouteWarps; ++w)
            s += red[w];
        p.losses[0] = s * float(E) / float(k) * inv;
        p.losses[1] = z * inv;
    }
}

// One warp a token:  d l_e = p_e (g_e - sum p g - sum_j [plain weights] p_j s dw_j + 2 dz lse / live) + add_e
// with p = exp(l - lse), g_e = dbal E c_e / (k live^2), and add the slots' own part:
// p_j s dw_j for plain weights, q_j s (dw_j - sum q dw) for normalised ones (q: softmax over the chosen).
template <class T, int V> __global__ void __launch_bounds__(kRouteThreads) route_grad(const RouteGradParams p) {
    extern __shared__ float grad_smem[];  // balance term [experts], then per warp the slots' part [experts]
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int E = p.experts, k = p.top_k;
    float *bal = grad_smem, *add = grad_smem + E * (1 + warp);
    const float n = float(max(*p.live, 1));
    const float db = p.dlosses ? p.dlosses[0] * float(E) / (float(k) * n * n) : 0.0f;
    const float dz = p.dlosses ? 2.0f * p.dlosses[1] / n : 0.0f;
    for (int e = threadIdx.x; e < E; e += kRouteThreads)
        bal[e] = db * float(p.counts[e]);
    for (int e = lane; e < E; e += 32)
        add[e] = 0.0f;
    __syncthreads();
    for (int64_t t = int64_t(blockIdx.x) * kRouteWarps + warp; t < p.tokens; t += int64_t(gridDim.x) * kRouteWarps) {
        T *out = static_cast<T *>(p.dlogits) + t * E;
        const float lse = p.lse[t];
        const bool there = (!p.mask || p.mask[t] != 0) && lse != -INFINITY;
        if (!there) {
            for (int e = lane; e < E; e += 32)
                out[e] = from_f32<T>(0.0f);
            continue;
        }
        const T *row = static_cast<const T *>(p.logits) + t * E;
        float v[V], dot = 0.0f;
        load_row<T, V>(v, row, E, true);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = expf(v[i] - lse);
            if (lane + 32 * i < E)
                dot += v[i] * bal[lane + 32 * i];
        }
        int id = -1;
        if (p.dweights && lane < k) {
            id = p.ids[t * k + lane];
            if (id < -1 || id >= E) {
                report(p.status, kSiteExpert);
                id = -1;
            }
        }
        if (p.dweights) {
            const float l = id >= 0 ? to_f32(row[id]) : -INFINITY;
            const float dw = id >= 0 ? p.dweights[t * k + lane] * p.scale : 0.0f;
            float mine;
            if (p.normalize) {
                float mx = l;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float ex = id >= 0 ? expf(l - mx) : 0.0f;
                const float sum = warp_sum(ex);
                const float q = id >= 0 ? ex / sum : 0.0f;
                mine = q * (dw - warp_sum(q * dw));
            } else {
                mine = id >= 0 ? expf(l - lse) * dw : 0.0f;
                dot += mine;
            }
            if (id >= 0)
                atomicAdd(&add[id], mine);  // one addend a place: a token's experts are distinct
        }
        dot = warp_sum(dot);
        __syncwarp();
        const float c = dz * lse - dot;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = lane + 32 * i;
            if (e < E)
                out[e] = from_f32<T>(v[i] * (bal[e] + c) + add[e]);
        }
        __syncwarp();
        if (id >= 0)
            add[id] = 0.0f;
        __syncwarp();
    }
}

}  // namespace moe
}  // namespace gg
