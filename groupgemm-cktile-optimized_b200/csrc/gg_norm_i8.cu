// Host side of the layer norm, its gradients, the rounding of rows to 8-bit integers and the 8-bit products: argument checks,
// workspaces and launches (C ABI in include/gg_b200.h).
#include <algorithm>
#include <cmath>

#include "gg_i8.cuh"
#include "gg_moe_host.h"
#include "gg_norm.cuh"

namespace {

using namespace gg::host;
using gg::fail;
using gg::MoeLaunch;
using gg::refuse;
using gg::moe::kNormFullThreads;
using gg::moe::kNormMaxGroups;
using gg::moe::kNormMaxHidden;
using gg::moe::kNormMaxSlots;
using gg::moe::kNormSmem;
using gg::moe::kNormThreads;

// ---- layer norm ----

struct NormShape {
    int v;  // vectors a thread
    bool full;
    int warps, groups, slots, params_at;
    unsigned blocks;
    size_t smem;
};

// full_threads: of a block of the check-free form, at most. ahead: bytes of rows that a block keeps on their way or in use, beyond the two that a
// group needs at least.
NormShape norm_shape(int64_t rows, int vecs, int v, int full_threads, int tensors, int elem, int params, int param_size, size_t ahead, int num_sms) {
    NormShape s{};
    s.v = v;
    s.warps = (vecs + 32 * s.v - 1) / (32 * s.v);
    s.full = s.v > 2 && vecs == 32 * s.v * s.warps;
    const int64_t each = (rows + num_sms - 1) / num_sms;  // rows of a block
    const size_t row = size_t(vecs) * 8 * size_t(elem) * size_t(tensors);
    int most = (s.full ? full_threads : kNormThreads) / (32 * s.warps);
    // what 768 threads add keeps to about `ahead` (7168 columns with a residual and 8-bit rows 191 us with a third group, 185 without)
    while (most > kNormThreads / (32 * s.warps) && size_t(most) * 2 * row > (100 << 10))
        --most;
    s.groups = int(std::max<int64_t>(1, std::min<int64_t>({each, most, kNormMaxGroups})));
    size_t copy = s.v > 2 ? size_t(params) * size_t(vecs) * 8 * size_t(param_size) : 0;
    if (2 * row + copy > size_t(kNormSmem))
        copy = 0;  // read from global memory
    while (s.groups > 1 && size_t(s.groups) * 2 * row + copy > size_t(kNormSmem))
        --s.groups;
    s.blocks = unsigned(std::min<int64_t>(num_sms, (rows + s.groups - 1) / s.groups));
    const int64_t turns = (each + s.groups - 1) / s.groups;  // rows of a group
    const int64_t fit = int64_t((kNormSmem - copy) / (size_t(s.groups) * row)), wanted = std::max<int64_t>(2, int64_t(ahead / (size_t(s.groups) * row)));
    s.slots = int(std::max<int64_t>(1, std::min<int64_t>({fit, wanted, turns, kNormMaxSlots})));
    s.smem = size_t(s.groups) * size_t(s.slots) * row;
    s.params_at = copy ? int(s.smem) : 0;
    s.smem += copy;
    return s;
}

template <class T, class W, int V, bool kFull> const void *norm_fn(bool grad) {
    return grad ? reinterpret_cast<const void *>(&gg::moe::norm_grad_rows<T, W, V, kFull>)
                : reinterpret_cast<const void *>(&gg::moe::norm_rows<T, W, V, kFull>);
}
template <class T, class W> const void *norm_fn(const NormShape &s, bool grad) {
    if (s.v == 1)
        return norm_fn<T, W, 1, false>(grad);
    if (s.v == 2)
        return norm_fn<T, W, 2, false>(grad);
    return s.full ? norm_fn<T, W, 4, true>(grad) : norm_fn<T, W, 4, false>(grad);
}
const void *norm_fn(const NormShape &s, int dtype, int param_type, bool grad) {
    if (dtype == GG_F32)
        return norm_fn<float, float>(s, grad);
    if (dtype == GG_FP16)
        return param_type == GG_F32 ? norm_fn<__half, float>(s, grad) : norm_fn<__half, __half>(s, grad);
    return param_type == GG_F32 ? norm_fn<__nv_bfloat16, float>(s, grad) : norm_fn<__nv_bfloat16, __nv_bfloat16>(s, grad);
}

const char *norm_bad(int32_t dtype, int32_t param_type, int64_t tokens, int64_t hidden) {
    if (dtype != GG_BF16 && dtype != GG_FP16 && dtype != GG_F32)
        return "dtype must be bf16 (0), fp16 (1) or fp32 (2)";
    if (param_type != dtype && param_type != GG_F32)
        return "param_type must be dtype or fp32 (2)";
    if (tokens < 0 || tokens >= kMaxIndex)
        return "tokens must be 0..2^31 - 1";
    if (hidden < 8 || hidden % 8 != 0 || hidden > kNormMaxHidden)
        return "hidden must be a multiple of 8 in 8..16384";
    return nullptr;
}

int prepare_norm(gg_handle *h, const gg_norm_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    if (const char *bad = norm_bad(q.dtype, q.param_type, q.tokens, q.hidden))
        return refuse(h, why, why_len, bad);
    if (!(q.eps >= 0.0f) || std::isinf(q.eps))
        return refuse(h, why, why_len, "eps must be finite and not negative");
    if (q.tokens > 0 && (!q.x || (!q.y && !q.q)))
        return refuse(h, why, why_len, "x and one of y and q must be non-null device pointers");
    if (!q.q != !q.q_scales)
        return refuse(h, why, why_len, "q and q_scales go together");
    if (q.sum && !q.residual)
        return refuse(h, why, why_len, "sum needs a residual");
    if (!aligned16({q.x, q.residual, q.gamma, q.beta, q.sum, q.y, q.q}) || !aligned4({q.mean, q.rstd, q.q_scales}))
        return refuse(h, why, why_len, "x, residual, gamma, beta, sum, y and q must be 16-byte aligned, the other operands 4-byte aligned");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    // Vectors a thread: as few warps a row as registers allow, which is two vectors, since the sums between lanes cost the same for any number; with
    // 8-bit rows, whose longer way wants two rows at a time, four.
    const int vecs = int(q.hidden / 8), v = vecs <= 64 ? 1 : vecs <= (q.q ? 96 : 1024) ? 2 : 4;
    const NormShape s = norm_shape(q.tokens, vecs, v, kNormFullThreads, q.residual ? 2 : 1, q.dtype == GG_F32 ? 4 : 2, 2, q.param_type == GG_F32 ? 4 : 2, 88 << 10, num_sms);
    gg::moe::NormParams p{};
    p.x = q.x;
    p.residual = q.residual;
    p.gamma = q.gamma;
    p.beta = q.beta;
    p.sum = q.sum;
    p.y = q.y;
    p.mean = q.mean;
    p.rstd = q.rstd;
    p.q = q.q;
    p.q_scales = q.q_scales;
    p.status = h->d_status;
    p.rows = q.tokens;
    p.vecs = vecs;
    p.warps = s.warps;
    p.groups = s.groups;
    p.slots = s.slots;
    p.params_at = s.params_at;
    p.eps = q.eps;
    p.timeout_ns = uint64_t(h->opt_timeout_ms) * 1000000u;
    p.test_stall = h->opt_test_stall;
    set_params(h, p);
    const void *fn = norm_fn(s, q.dtype, q.param_type, false);
    GG_CUDA(h, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmem));
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_norm<%s> hidden=%lld blocks=%u groups=%d warps=%d slots=%d", type_name(q.dtype),
                  static_cast<long long>(q.hidden), s.blocks, s.groups, s.warps, s.slots);
    return finish(h, stream, {MoeLaunch{fn, s.blocks, unsigned(s.groups * s.warps * 32), s.smem}}, detail);
}

int prepare_norm_grad(gg_handle *h, const gg_norm_grad_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    if (const char *bad = norm_bad(q.dtype, q.param_type, q.tokens, q.hidden))
        return refuse(h, why, why_len, bad);
    if (q.tokens > 0 && (!q.x || !q.mean || !q.rstd || !q.dy || !q.dx))
        return refuse(h, why, why_len, "x, mean, rstd, dy and dx must be non-null device pointers");
    if (!aligned16({q.x, q.gamma, q.dy, q.dsum, q.dx}) || !aligned4({q.mean, q.rstd, q.dgamma, q.dbeta}))
        return refuse(h, why, why_len, "x, gamma, dy, dsum and dx must be 16-byte aligned, the other operands 4-byte aligned");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    const int vecs = int(q.hidden / 8), v = vecs <= 64 ? 1 : vecs <= 512 ? 2 : 4;
    const NormShape s = norm_shape(q.tokens, vecs, v, kNormThreads, q.dsum ? 3 : 2, q.dtype == GG_F32 ? 4 : 2, 1, q.param_type == GG_F32 ? 4 : 2, 160 << 10, num_sms);
    const size_t sums = 2 * size_t(q.hidden) * 4;  // dgamma and dbeta of a block or group
    if (const int rc = reserve(h, std::max<size_t>(1, s.blocks) * sums))
        return rc;
    gg::moe::NormGradParams p{};
    p.x = q.x;
    p.dy = q.dy;
    p.dsum = q.dsum;
    p.gamma = q.gamma;
    p.mean = q.mean;
    p.rstd = q.rstd;
    p.dx = q.dx;
    p.dgamma = q.dgamma;
    p.dbeta = q.dbeta;
    p.parts = h->d_ws;
    p.status = h->d_status;
    p.rows = q.tokens;
    p.vecs = vecs;
    p.warps = s.warps;
    p.groups = s.groups;
    p.slots = s.slots;
    p.params_at = s.params_at;
    p.blocks = int(s.blocks);
    p.timeout_ns = uint64_t(h->opt_timeout_ms) * 1000000u;
    p.test_stall = h->opt_test_stall;
    set_params(h, p);
    const void *fn = norm_fn(s, q.dtype, q.param_type, true);
    GG_CUDA(h, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmem));
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_norm_grad<%s> hidden=%lld blocks=%u groups=%d warps=%d slots=%d", type_name(q.dtype),
                  static_cast<long long>(q.hidden), s.blocks, s.groups, s.warps, s.slots);
    const MoeLaunch rows{fn, s.blocks, unsigned(s.groups * s.warps * 32), std::max(s.smem, size_t(s.groups - 1) * sums)};
    const MoeLaunch sum{reinterpret_cast<const void *>(&gg::moe::norm_grad_sum), q.dgamma || q.dbeta ? unsigned((2 * q.hidden + 31) / 32) : 0u,
                        gg::moe::kNormSumWarps * 32, 0};
    return finish(h, stream, {rows, sum}, detail);
}

// ---- rounding to 8-bit integers ----

const void *quant_fn(int dtype) {
    return dtype == GG_F32    ? reinterpret_cast<const void *>(&gg::moe::quant_rows<float>)
           : dtype == GG_FP16 ? reinterpret_cast<const void *>(&gg::moe::quant_rows<__half>)
                              : reinterpret_cast<const void *>(&gg::moe::quant_rows<__nv_bfloat16>);
}

// Threads of a block that rounds rows of k.
unsigned quant_threads(int64_t rows, int64_t k, int num_sms) {
    const int64_t vecs = k / 8, each = rows > 4 * num_sms ? gg::moe::kQuantHeld : 1;
    return unsigned(std::min<int64_t>(512, ((vecs + each - 1) / each + 31) / 32 * 32));
}

int prepare_quant(gg_handle *h, const gg_quant_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    if (q.dtype != GG_BF16 && q.dtype != GG_FP16 && q.dtype != GG_F32)
        return refuse(h, why, why_len, "dtype must be bf16 (0), fp16 (1) or fp32 (2)");
    if (q.rows < 0 || q.rows >= kMaxIndex)
        return refuse(h, why, why_len, "rows must be 0..2^31 - 1");
    if (q.k < 8 || q.k % 8 != 0 || q.k > (int64_t(1) << 30))
        return refuse(h, why, why_len, "k must be a multiple of 8 (16-byte rows) in 8..2^30");
    if (q.rows > 0 && (!q.x || !q.q || !q.scales))
        return refuse(h, why, why_len, "x, q and scales must be non-null device pointers");
    if (!aligned16({q.x, q.q}) || !aligned4({q.scales}))
        return refuse(h, why, why_len, "x and q must be 16-byte aligned, scales 4-byte aligned");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    gg::moe::QuantParams p{q.x, q.q, q.scales, q.rows, int(q.k / 8)};
    set_params(h, p);
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_quant<%s> k=%lld", type_name(q.dtype), static_cast<long long>(q.k));
    const MoeLaunch rows{quant_fn(q.dtype), unsigned(std::min<int64_t>(q.rows, 32 * num_sms)), quant_threads(q.rows, q.k, num_sms), 0};
    return finish(h, stream, {rows}, detail);
}

// ---- 8-bit products ----

template <class T> const void *i8_products_fn(bool once) {
    return once ? reinterpret_cast<const void *>(&gg::moe::i8_products<T, true>) : reinterpret_cast<const void *>(&gg::moe::i8_products<T, false>);
}

int prepare_i8(gg_handle *h, const gg_i8_problem &q, gg_stream_t stream, char *why, size_t why_len) {
    using namespace gg::moe;
    if (q.dtype != GG_BF16 && q.dtype != GG_FP16)
        return refuse(h, why, why_len, "dtype must be bf16 (0) or fp16 (1)");
    if (q.experts < 1 || q.experts > kI8MaxExperts)
        return refuse(h, why, why_len, "experts must be 1..1024");
    if (q.n < 8 || q.n % 8 != 0 || q.n > (int64_t(1) << 30))
        return refuse(h, why, why_len, "n must be a multiple of 8 (16-byte output row stride) in 8..2^30");
    if (q.k < 16 || q.k % 16 != 0 || q.k > kI8MaxK)
        return refuse(h, why, why_len, "k must be a multiple of 16 (16-byte rows) in 16..131056 (sums in 32 bits)");
    if (q.rows < 0 || q.rows >= kMaxIndex)
        return refuse(h, why, why_len, "rows must be 0..2^31 - 1");
    if (q.src && (q.tokens < 0 || q.tokens >= kMaxIndex || q.top_k < 1 || q.tokens * q.top_k >= kMaxIndex))
        return refuse(h, why, why_len, "with src, tokens must be >= 0, top_k >= 1 and tokens * top_k below 2^31");
    if (q.src && q.tokens == 0 && q.rows > 0)
        return refuse(h, why, why_len, "rows without tokens");
    if (!q.offsets || !q.weight || !q.scales || (q.rows > 0 && (!q.x || !q.out)))
        return refuse(h, why, why_len, "x, weight, scales, offsets and out must be non-null device pointers");
    if (!aligned16({q.x, q.weight, q.out}) || !aligned4({q.x_scales, q.scales, q.offsets, q.src}))
        return refuse(h, why, why_len, "x, weight and out must be 16-byte aligned, x_scales, scales, offsets and src 4-byte aligned");
    if (q.n * q.k >= int64_t(1) << 39)
        return refuse(h, why, why_len, "one expert's weights are too large for a TMA descriptor");
    const int64_t tiles = (q.n + kI8TileRows - 1) / kI8TileRows, steps = (q.k + kI8StepK - 1) / kI8StepK;
    if (std::min(q.rows, q.experts + q.rows / 32) * tiles >= kMaxIndex)
        return refuse(h, why, why_len, "too many weight rows and experts for one launch");
    int num_sms = 0;
    if (const int rc = bind_device(h, stream, num_sms, why, why_len))
        return rc;
    const int pairs = num_sms / 2;
    // Tokens of a chunk at most: a stage has place for half of them beside its 16 KB of weights, so that small chunks keep more weights on
    // their way, but an expert with more rows than that has its weights loaded again. And chunks small enough that there are about as many
    // items as pairs, before any are cut along k. `once`: weights leave L2 first. Us with chunks of 64 / 128 / 256, and in brackets once, of
    // 32 experts of 4096 x 4096 by their mean rows: 8 87 (83) / 87 (83) / 87 (84); 32 91 (86) / 91 (88) / 94 (90); 48 100 (97) / 97 (94) / 97 (93);
    // 64 100 (99) / 96 (93) / 99 (95); 96 119 (121) / 102 (103) / 103 (101); 128 142 (149) / 116 (118) / 111 (111); 256 234 (241) / 173 (177) / 147 (151).
    // All for even loads: the host does not see the counts, so rows that all go to few of many experts take the chunks of their mean (1024 rows of
    // one of 64 experts of 4096 x 7168 56 us, with chunks of 256 32; 900 of one and 2 of each other 316 and 309).
    const int64_t mean = q.rows / q.experts;
    int chunk = mean <= 32 ? 64 : mean <= 64 ? 128 : kI8MaxTokens;
    while (chunk > 32 && (q.rows + chunk / 2 - 1) / (chunk / 2) * tiles <= pairs)
        chunk /= 2;
    const bool order = q.rows > 0 && (q.src || !q.x_scales);  // rows are put into expert order or rounded first
    const size_t sums = 2 * size_t(pairs) * size_t(chunk) * 1024, rounded = order ? size_t(q.rows) * size_t(q.k) : 0;
    // By tokens where a token has several places and there is more to move than the launch before costs: us by places / by tokens, 1024 x 8 rows
    // of 7168 291 / 293, 2048 x 8 of 4096 97.5 / 96.8, 16384 x 2 of 7168 777 / 734 (with the products). Where there are fewer rows than slots
    // (other experts' are elsewhere), tokens without a place are read for nothing: 65536 tokens of 2880 in 16 bits with 1/8, 1, 1.25, 1.5 and 2
    // rows a token 31 / 127, 169 / 191, 209 / 208, 248 / 224 and 320 / 253, 16384 of 4096 in 8 bits with 1, 1.5 and 2 40 / 47, 60 / 64 and 72 / 73
    // (both with 8 weight rows only).
    const bool by_token = order && q.src && q.top_k >= 2 && q.top_k <= kI8TokenPlaces && q.rows * q.k >= int64_t(1) << 23 &&
                          8 * q.rows >= (q.x_scales ? 15 : 10) * q.tokens;
    if (const int rc = reserve(h, sums + rounded + (order ? size_t(q.rows) * 4 : 0) + (by_token ? size_t(q.tokens) * size_t(q.top_k) * 4 : 0)))
        return rc;
    if (const int rc = reserve_counters(h, size_t(pairs) * 2 * kI8EpilogueWarps * 4, stream))
        return rc;
    I8Params p{};
    p.x = q.x;
    p.x_scales = q.x_scales;
    p.xq = order ? reinterpret_cast<int8_t *>(h->d_ws) + sums : static_cast<int8_t *>(const_cast<void *>(q.x));
    p.xq_scales = order ? reinterpret_cast<float *>(p.xq + rounded) : const_cast<float *>(q.x_scales);
    p.inv = by_token ? reinterpret_cast<int32_t *>(p.xq_scales + q.rows) : nullptr;
    p.scales = q.scales;
    p.offsets = q.offsets;
    p.src = q.src;
    p.out = q.out;
    p.status = h->d_status;
    p.ws = reinterpret_cast<int32_t *>(h->d_ws);
    p.counters = h->d_counters;
    p.rows = q.rows;
    p.slots = q.src ? q.tokens * q.top_k : 0;
    p.timeout_ns = uint64_t(h->opt_timeout_ms) * 1000000u;
    p.test_stall = h->opt_test_stall;
    p.n = int(q.n);
    p.k = int(q.k);
    p.experts = q.experts;
    p.top_k = q.src ? q.top_k : 1;
    p.tiles = int(tiles);
    p.steps = int(steps);
    p.chunk = chunk;
    p.stage_bytes = kI8WeightBytes + chunk / 2 * kI8StepK;
    p.stages = std::min(kI8MaxStages, kI8Ring / p.stage_bytes);
    p.after_rows = order ? 1 : 0;
    if (q.rows > 0) {
        if (const int rc = encode_bytes_3d(h, h->moe.map[0], q.weight, q.k, q.n, q.experts, kI8StepK, kI8TileRows / 2, CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
        if (const int rc = encode_bytes_2d(h, h->moe.map[1], p.xq, q.k, q.rows, kI8StepK, unsigned(chunk / 2), CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
    }
    set_params(h, p);
    const bool half = q.dtype == GG_FP16;
    const void *fn = half ? i8_products_fn<__half>(mean <= 128) : i8_products_fn<__nv_bfloat16>(mean <= 128);
    GG_CUDA(h, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kI8Smem));
    const void *rows_fn = by_token ? (half ? reinterpret_cast<const void *>(&i8_token_rows<__half>) : reinterpret_cast<const void *>(&i8_token_rows<__nv_bfloat16>))
                                   : (half ? reinterpret_cast<const void *>(&i8_rows<__half>) : reinterpret_cast<const void *>(&i8_rows<__nv_bfloat16>));
    const int64_t sources = by_token ? q.tokens : q.rows;
    const MoeLaunch places{reinterpret_cast<const void *>(&i8_places),
                           by_token ? unsigned(std::min<int64_t>((q.rows + kI8PlaceThreads - 1) / kI8PlaceThreads, 8 * num_sms)) : 0u, kI8PlaceThreads, 0};
    const MoeLaunch rows{rows_fn, order ? unsigned(std::min<int64_t>(sources, 32 * num_sms)) : 0u,
                         quant_threads(sources, q.x_scales ? q.k / 2 : q.k, num_sms), 0};
    MoeLaunch products{fn, q.rows > 0 ? unsigned(2 * pairs) : 0u, kI8Threads, size_t(kI8Smem), 2};
    products.cluster = 2;
    char detail[160];
    std::snprintf(detail, sizeof(detail), "gg_i8<%s> n=%lld k=%lld chunk=%d stages=%d pairs=%d", type_name(q.dtype), static_cast<long long>(q.n),
                  static_cast<long long>(q.k), chunk, p.stages, pairs);
    return finish(h, stream, {places, rows, products}, detail);
}

}  // namespace

extern "C" {

int gg_prepare_norm(gg_handle *h, const gg_norm_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_norm(h, *p, stream, why, why_len);
    });
}

int gg_prepare_norm_grad(gg_handle *h, const gg_norm_grad_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_norm_grad(h, *p, stream, why, why_len);
    });
}

int gg_prepare_quant(gg_handle *h, const gg_quant_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_quant(h, *p, stream, why, why_len);
    });
}

int gg_prepare_i8(gg_handle *h, const gg_i8_problem *p, gg_stream_t stream, char *why, size_t why_len) {
    return guarded(h, [&] {
        if (const int rc = begin(h, p, why, why_len))
            return rc;
        return prepare_i8(h, *p, stream, why, why_len);
    });
}

}  // extern "C"
