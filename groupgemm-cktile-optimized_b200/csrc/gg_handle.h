// The handle behind the C ABI of include/gg_b200.h, and the error helpers its entry points share.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <string>

#include "gg_b200.h"
#include "gg_kernel.cuh"

namespace gg {

// One kernel of a prepared layer operator (router, dispatch / combine, norm, 4- and 8-bit products):
// gg_run launches them in order, each with the operator's parameter block as its argument (after the
// tensor maps where it has some). A kernel may take a part of the block that stands first in it.
struct MoeLaunch {
    const void *fn = nullptr;
    unsigned grid = 0, block = 0;
    size_t smem = 0;
    int maps = 0;  // the kernel takes MoePlan::map[0 .. maps) first
    unsigned grid_y = 1, cluster = 1;  // cluster: blocks of one along x
};

struct MoePlan {
    int launches = 0;  // 0: the handle holds no layer operator
    MoeLaunch launch[3];
    CUtensorMap map[2]{};
    alignas(16) unsigned char params[256];
};

// Enqueues the handle's prepared layer operator (gg_moe.cu).
int run_moe(gg_handle *h, cudaStream_t stream);

}  // namespace gg

struct gg_handle {
    // options
    int opt_variant = -1;
    int opt_band = 0;
    int opt_raster = -1;
    int opt_bn = 0;
    int opt_split = 0;
    int opt_sk_tail = -1;
    int opt_stream_k = 0;  // 0 off (default), -1 cost model decides, 1 / 2 stream-K over the partial
                           // last wave (+ one wave)
    int opt_max_ctas = 0;
    int64_t opt_timeout_ms = 2000;
    int opt_test_stall = 0;
    int opt_test_bounds = 0;  // test only: declare the output one row short to the debug build's checks
    int opt_pdl = 1;
    int opt_store = -1;  // -1 auto, 0 = staging + TMA stores, 1 = direct stores
    int opt_tail = -1;   // split launch for skewed routing: -1 auto, 0 off, 1 on
    int opt_chunks = 1;  // wgrad: 3-D chunk views for the MN-major operand loads where the shape allows
    int opt_order = 0;  // planned tile order (wgrad with store-bound and tensor-bound groups): -1 auto, 0 off, 1 on
    int opt_half = 0;    // 1 on (half-height last tiles where a group allows), 0 off (default), -1 = on
    int opt_sched = 0;  // -1 auto (dynamic for multi-wave launches of whole tiles), 0 static, 1 dynamic
    int opt_l2_a = -1;  // L2 eviction priority of the A / B operand loads (forward):
    int opt_l2_b = 0;   // 0 no hint, 1 evict_first, 2 evict_last; l2_a -1 = automatic

    // prepared state
    bool ready = false;
    int device = -1;
    int dtype = 0;
    int variant = 0;
    int64_t total_m = 0;
    int32_t *d_meta = nullptr;  // tile_off[G+1] then row_off[G+1]
    size_t meta_cap = 0;        // int32 entries
    uint32_t *d_status = nullptr;
    float *d_ws = nullptr;  // split-K partial sums
    size_t ws_cap = 0;      // bytes
    int32_t *d_counters = nullptr;
    size_t counters_cap = 0;  // bytes
    int32_t *d_tiles = nullptr;      // planned tile order: (group, mt << 16 | nt) per tile
    size_t tiles_cap = 0;            // int32 entries
    CUtensorMap *d_gmaps = nullptr;  // wgrad: per-group tensor maps
    size_t gmaps_cap = 0;            // maps
    int op = 0;                      // gg::kOpForward / kOpDgrad / kOpWgrad
    CUtensorMap tmap_a{}, tmap_b{}, tmap_out{};
    CUtensorMap tmap_a_half{};  // A in 64-row boxes, for half-height pair tiles
    // Second launch of a split launch: the one-CTA kernel over the groups' remainders of at most
    // 128 rows (tmap_a / tmap_out are shared with the first launch).
    struct {
        bool active = false;
        const void *fn = nullptr;
        int grid = 0, smem = 0;
        CUtensorMap tmap_b{};
        gg::KernelParams params{};
    } tail;
    gg::KernelParams params{};
    int grid = 0;
    const void *fn = nullptr;
    int smem = 0;
    int cg = 1;

    gg::MoePlan moe;  // a prepared layer operator, or none: then the fields above hold a grouped GEMM

    std::string detail, last_error;
};

namespace gg {

inline int fail(gg_handle *h, int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    h->last_error = buf;
    return code;
}

inline int refuse(gg_handle *h, char *why, size_t why_len, const char *msg) {
    h->last_error = msg;
    if (why && why_len > 0) {
        std::strncpy(why, msg, why_len - 1);
        why[why_len - 1] = '\0';
    }
    return GG_NOT_SUPPORTED;
}

#define GG_CUDA(h, expr)                                                                                  \
    do {                                                                                                  \
        cudaError_t e_ = (expr);                                                                          \
        if (e_ != cudaSuccess)                                                                            \
            return gg::fail((h), GG_ERR_CUDA, "%s: %s (%s:%d)", #expr, cudaGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)

}  // namespace gg
