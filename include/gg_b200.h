/*
 * gg_b200.h — C ABI of the B200 (sm_100a) grouped-GEMM backend.
 *
 * Operation (forward MoE grouped GEMM, RCR layout), the op of the reference's
 * GroupedGemmProblem (common/backend.hpp:32-60):
 *
 *     out[rows of group g] = x[rows of group g] @ w[g]^T
 *     x   [sum(group_m), k]  row-major   (tokens of all experts, back to back)
 *     w   [group_num, n, k]  row-major   (one weight matrix per expert)
 *     out [sum(group_m), n]  row-major
 *     bf16 or fp16 in, fp32 accumulation, output in the input dtype.
 *
 * The entry points mirror the reference's `class Backend` (common/backend.hpp:62-79):
 * prepare() is untimed set-up that returns "" or a reason the shape cannot run, run() enqueues
 * exactly one grouped GEMM without synchronising, release() frees what prepare() allocated.
 * Instead of exiting on a device error (TUNEMAX_HIP_CHECK, common/backend.hpp:15-23) every call
 * returns a status code and the library never terminates the process.
 *
 * Plain pointers and sizes only. `gg_stream_t` is the same type as CUDA's cudaStream_t
 * (NULL = the legacy default stream). A handle is bound to the device that is current when
 * gg_prepare() is called; it is not thread-safe (one handle per thread and device).
 */
#ifndef GG_B200_H
#define GG_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st *gg_stream_t; /* == cudaStream_t */
typedef struct gg_handle gg_handle;

/* Element types (tunemax::DType, common/backend.hpp:27). */
enum gg_dtype { GG_BF16 = 0, GG_FP16 = 1, GG_F32 = 2 /* router logits, norm, rounding to 8 bits */ };

/* Return codes. */
enum gg_status {
    GG_OK = 0,            /* ready / done */
    GG_NOT_SUPPORTED = 1, /* gg_prepare: shape or arguments refused; `why` holds the reason (N/A) */
    GG_ERR_ARG = -1,      /* invalid call (null handle, run before prepare, ...) */
    GG_ERR_CUDA = -2,     /* a CUDA runtime/driver call failed; see gg_last_error() */
    GG_ERR_DEVICE = -3    /* the kernel reported a bounded-wait timeout; see gg_device_status() */
};

/* Problem descriptor: tunemax::GroupedGemmProblem (common/backend.hpp:39-60). group_m is a host
 * array of group_num entries (any value >= 0; zero-length groups are skipped); x, w, out are
 * device pointers owned by the caller, 16-byte aligned. Requirements checked by gg_prepare:
 * k % 8 == 0 and n % 8 == 0 (16-byte row strides for TMA and the vector epilogue),
 * sum(group_m) < 2^31. */
typedef struct gg_problem {
    int32_t dtype;          /* enum gg_dtype */
    int32_t group_num;      /* B: number of groups (experts) */
    int64_t n;              /* N: output columns = rows of each w[g] */
    int64_t k;              /* K: reduction length */
    const int64_t *group_m; /* host, [group_num] rows per group */
    const void *x;          /* device, [sum(group_m), k] */
    const void *w;          /* device, [group_num, n, k] */
    void *out;              /* device, [sum(group_m), n] */
} gg_problem;

/* Create a backend instance (tunemax::make_ck_tile_backend(), common/backend.hpp:81, is the
 * factory this one sits beside). Returns NULL only when out of host memory. */
gg_handle *gg_create(void);

/* Backend::name() (common/backend.hpp:65). Returns "b200". */
const char *gg_name(const gg_handle *h);

/* Backend::prepare() (common/backend.hpp:66; the CK version is ck_kernel/ck_grouped_gemm.cpp:
 * 130-218). Untimed: validates the problem, builds the device group-argument buffer (per-group
 * tile and row offsets), encodes the TMA descriptors and picks the kernel variant, then waits
 * for `stream`. Returns GG_OK when ready, GG_NOT_SUPPORTED with a reason in `why` (if why != NULL
 * and why_len > 0) when the shape is refused, or a negative error. */
int gg_prepare(gg_handle *h, const gg_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Backward grouped GEMMs of the same layer (MoE training). The reference benchmarks the forward
 * op only; its vendored Primus-Turbo grouped GEMM carries the two backward calls this replaces
 * (third_party/primus_turbo/kernels/hipblaslt_grouped_gemm.cu:80-96 shape rules,
 * :199-240 per-group arguments, zero-filled gradient for an expert without tokens :201-214):
 *
 *   GG_OP_DGRAD: dx[rows of g] = dy[rows of g] @ w[g]     dx [sum(group_m), k]
 *   GG_OP_WGRAD: dw[g] = dy[rows of g]^T @ x[rows of g]   dw [group_num, n, k]; an expert with
 *                                                         group_m[g] == 0 gets dw[g] = 0
 *
 * with dy [sum(group_m), n] (the gradient of out), x and w as in gg_problem. Same dtype rules,
 * fp32 accumulation, output in the input dtype (dw is overwritten, not accumulated into). */
enum gg_op { GG_OP_FORWARD = 0, GG_OP_DGRAD = 1, GG_OP_WGRAD = 2 };

typedef struct gg_grad_problem {
    int32_t dtype;          /* enum gg_dtype */
    int32_t group_num;      /* B */
    int64_t n;              /* N: columns of dy = rows of each w[g] */
    int64_t k;              /* K: columns of x, dx and each w[g] */
    const int64_t *group_m; /* host, [group_num] tokens per group */
    const void *dy;         /* device, [sum(group_m), n] */
    const void *x;          /* device, [sum(group_m), k]  (GG_OP_WGRAD) */
    const void *w;          /* device, [group_num, n, k]  (GG_OP_DGRAD) */
    void *dx;               /* device, [sum(group_m), k]  (GG_OP_DGRAD output) */
    void *dw;               /* device, [group_num, n, k]  (GG_OP_WGRAD output) */
} gg_grad_problem;

/* Backend::prepare() for a backward operation `op` (GG_OP_DGRAD or GG_OP_WGRAD); afterwards
 * gg_run() enqueues it as one kernel launch and gg_detail() describes it. The operands the
 * operation does not use may be NULL. Extra refusals: "split" > 1 for wgrad (its reduction
 * length differs per group), group_num * n >= 2^31 for wgrad, and a forced "bn" that is not a
 * multiple of 64 per CTA (the MN-major operand boxes are 64 columns wide). */
int gg_prepare_grad(gg_handle *h, const gg_grad_problem *p, int32_t op, gg_stream_t stream, char *why,
                    size_t why_len);

/* ---- The layer around the grouped GEMM ----
 *
 * Router, token movement, norm, and 4- and 8-bit products of the same mixture-of-experts layer. The reference
 * benchmarks the grouped GEMM alone, on rows that are in expert order already; these calls produce
 * that order, take the rows there and back, and serve few tokens from small weights. Each prepare
 * call below is used as gg_prepare: it validates (GG_NOT_SUPPORTED with a reason in `why`), allocates
 * what the handle needs and waits for `stream`; then gg_run() enqueues the operator on any stream
 * without waiting and allocates nothing (it can be captured in a CUDA graph; what was captured is good
 * until the handle is prepared again or released, either of which may free memory that it uses). A
 * handle holds one prepared operator at a time and its launches must not overlap on the GPU. Operands are device
 * pointers to contiguous arrays that the caller owns; the contents may change between runs.
 *
 * Indices that come from device memory (dest, src, ids, offsets) are checked by the kernels: one
 * that is out of range is skipped and reported by gg_device_status (GG_ERR_DEVICE, status
 * 0x2000 | site: 0x10 dest, 0x11 src, 0x12 offsets, 0x13 ids); nothing is read or written out of
 * bounds. Sums and softmax statistics are held in fp32; results do not depend on the order in which
 * the GPU runs blocks (the same inputs give the same bits). */

/* Router. For each token t with logits l_t [experts]:
 *
 *   lse_t = log sum_e exp(l_te)        p_te = exp(l_te - lse_t)
 *   ids_t: the top_k largest logits, falling, ties to the lower expert; -1 where fewer than top_k
 *          logits are above -inf (an expert at -inf is closed to the token)
 *   weights_tj = scale * p_t,ids_tj, or with `normalize` scale * exp(l_t,ids_tj) / sum_i exp(l_t,ids_ti);
 *          0 where ids is -1
 *
 * A token whose mask byte is 0, or all of whose logits are -inf, is not live: ids -1, weights 0, lse -inf,
 * and nothing of its logits (NaN included) goes anywhere. In a live row NaN counts as larger than +inf for
 * the choice, and a row that holds NaN or +inf has NaN weights and lse (as the formulas give).
 * With u = 2^-24 and d a logit's distance from the row's largest, a probability's relative error is up to (2 d + 64) u, and
 * one below 2^-126 of the largest counts as 0; lse's error is that of one rounding and of the sum, (|lse| + 64) u at most.
 *
 *   counts_e: slots (t, j) of expert e       offsets: their exclusive prefix sums, [experts + 1]
 *   dest_tj: place of slot (t, j) in the order by expert, slots of one expert in (t, j) order; -1 for none
 *   src: the slot t * top_k + j at each place, -1 from offsets[experts] on
 *   live: number of live tokens
 *   prob_e = (1 / live) sum_t p_te
 *   losses[0] = experts * sum_e counts_e / (top_k live) * prob_e        (balance loss)
 *   losses[1] = (1 / live) sum_t lse_t^2                                (z loss); both 0 if live is 0
 *
 * experts 1..1024, top_k 1..32 (at most experts), tokens * top_k < 2^31; logits 16-byte aligned. */
typedef struct gg_route_problem {
    int32_t logits_type;  /* GG_BF16, GG_FP16 or GG_F32 */
    int32_t experts;
    int32_t top_k;
    int32_t normalize;    /* 0 or 1 */
    float scale;          /* factor of the weights, 1 for none */
    int64_t tokens;       /* >= 0 */
    const void *logits;   /* [tokens, experts] */
    const uint8_t *mask;  /* [tokens], 0 = padding token; or NULL */
    int32_t *ids;         /* out [tokens, top_k] */
    float *weights;       /* out [tokens, top_k] */
    float *lse;           /* out [tokens], or NULL (gg_prepare_route_grad needs it) */
    int32_t *counts;      /* out [experts] */
    int32_t *offsets;     /* out [experts + 1] */
    int32_t *live;        /* out [1] */
    int32_t *dest;        /* out [tokens, top_k] */
    int32_t *src;         /* out [tokens * top_k] */
    float *prob;          /* out [experts], or NULL */
    float *losses;        /* out [2], or NULL */
} gg_route_problem;

int gg_prepare_route(gg_handle *h, const gg_route_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Gradient of the router's weights and losses with respect to the logits, from what gg_prepare_route's
 * run wrote (ids, lse, counts, live) and the same logits, mask, normalize and scale. counts are constants
 * of the balance loss, as usual. dweights or dlosses may be NULL (zero). Tokens that are not live and
 * closed experts get zero; what dweights holds at slots without an expert is not read. */
typedef struct gg_route_grad_problem {
    int32_t logits_type;
    int32_t experts;
    int32_t top_k;
    int32_t normalize;
    float scale;
    int64_t tokens;
    const void *logits;     /* [tokens, experts] */
    const uint8_t *mask;    /* [tokens] or NULL */
    const int32_t *ids;     /* [tokens, top_k] */
    const float *lse;       /* [tokens] */
    const int32_t *counts;  /* [experts] */
    const int32_t *live;    /* [1] */
    const float *dweights;  /* [tokens, top_k] or NULL */
    const float *dlosses;   /* [2]: of the balance and of the z loss; or NULL */
    void *dlogits;          /* out [tokens, experts], type of the logits */
} gg_route_grad_problem;

int gg_prepare_route_grad(gg_handle *h, const gg_route_grad_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Tokens into expert order and back, over the places `dest` that the router gives:
 *
 *   GG_OP_DISPATCH:     rows[dest_tj] = x_t; rows from offsets[experts] on are zero
 *   GG_OP_COMBINE:      x_t = sum_j weights_tj * rows[dest_tj] (fp32 sum; weights NULL = 1, which is the
 *                       gradient of dispatch)
 *   GG_OP_COMBINE_GRAD: drows[dest_tj] = weights_tj * dy_t (rows from offsets[experts] on are zero) and
 *                       dweights_tj = <dy_t, rows[dest_tj]> (0 without a place; dweights may be NULL)
 *
 * bf16 or fp16, hidden a multiple of 8, rows [tokens * top_k, hidden], 16-byte aligned; dest's entries
 * distinct, as the router's are. */
enum gg_permute_op { GG_OP_DISPATCH = 3, GG_OP_COMBINE = 4, GG_OP_COMBINE_GRAD = 5 };

typedef struct gg_permute_problem {
    int32_t dtype;
    int32_t experts;         /* length of offsets - 1 */
    int32_t top_k;
    int64_t tokens;
    int64_t hidden;
    void *x;                 /* [tokens, hidden]: read by dispatch, written by combine */
    void *rows;              /* [tokens * top_k, hidden]: written by dispatch, else read */
    const void *dy;          /* [tokens, hidden] (combine_grad) */
    void *drows;             /* out [tokens * top_k, hidden] (combine_grad) */
    const int32_t *dest;     /* [tokens, top_k] */
    const int32_t *offsets;  /* [experts + 1] (dispatch, combine_grad) */
    const float *weights;    /* [tokens, top_k], or NULL = 1 */
    float *dweights;         /* out [tokens, top_k] (combine_grad), or NULL */
} gg_permute_problem;

int gg_prepare_permute(gg_handle *h, const gg_permute_problem *p, int32_t op, gg_stream_t stream, char *why, size_t why_len);

/* Products with 4-bit weights for few rows an expert (decoding):
 *
 *   out[r, n] = sum over groups g of scales[e, n, g] * sum_{k in g} (q[e, n, k] - zeros[e, n, g]) * x[row(r), k]
 *
 * for the rows r of expert e, offsets[e] <= r < offsets[e + 1]; row(r) = src[r] / top_k, or r without
 * src (so the first product of a layer gathers its tokens itself). Rows of no expert are zero, and all rows where offsets
 * fall (which is reported). offsets and src are the router's, in device memory: no count goes to the host. q is 4 bits, two to a byte (even k in the low
 * half), zeros NULL = 8 everywhere (else its low four bits). The integers q - zero are exact in 16 bits,
 * products are summed in fp32, the scale is applied to each group's fp32 sum, and the result rounded once.
 *
 * bf16 or fp16 x, scales and out; experts 1..1024, n a multiple of 8, k a multiple of 32 (the last group
 * may be shorter), group_size 32, 64 or 128; x, qweight, scales, zeros and out 16-byte aligned. */
typedef struct gg_w4_problem {
    int32_t dtype;
    int32_t experts;
    int32_t group_size;
    int32_t top_k;           /* with src */
    int64_t n;
    int64_t k;
    int64_t rows;            /* rows of out */
    int64_t tokens;          /* rows of x, with src */
    const void *x;           /* [tokens, k] with src, else [rows, k] */
    const void *qweight;     /* [experts, n, k / 2] bytes */
    const void *scales;      /* [experts, n, ceil(k / group_size)] */
    const void *zeros;       /* [experts, n, ceil(k / group_size)] bytes, or NULL */
    const int32_t *offsets;  /* [experts + 1] */
    const int32_t *src;      /* [rows] or NULL */
    void *out;               /* [rows, n] */
} gg_w4_problem;

int gg_prepare_w4(gg_handle *h, const gg_w4_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Layer norm of each token, in front of the layer, with the residual that it is added to:
 *
 *   s = x + residual, rounded to dtype (or x)      mean_t = mean of s_t      rstd_t = 1 / sqrt(mean of (s_t - mean_t)^2 + eps)
 *   y = (s - mean) * rstd * gamma + beta           sum = s
 *   q, q_scales: y rounded to 8-bit integers as gg_prepare_quant does, in the same pass (for gg_prepare_i8)
 *
 * dtype bf16, fp16 or fp32 (x, residual, sum, y); param_type that or GG_F32 (gamma, beta). Statistics are fp32, of the squares
 * around the mean: a row whose squares pass fp32's largest value has rstd 0 and y = beta, one whose sum (or that of a part of its columns)
 * does NaN. sum may be the same array as x or residual, y the same as x where sum is not asked for. hidden a multiple of 8 up to 16384; x, residual, gamma, beta,
 * sum, y and q 16-byte aligned. */
typedef struct gg_norm_problem {
    int32_t dtype;
    int32_t param_type;      /* of gamma and beta */
    float eps;               /* >= 0 */
    int64_t tokens;
    int64_t hidden;
    const void *x;           /* [tokens, hidden] */
    const void *residual;    /* [tokens, hidden] or NULL */
    const void *gamma;       /* [hidden], or NULL = 1 */
    const void *beta;        /* [hidden], or NULL = 0 */
    void *sum;               /* out [tokens, hidden], or NULL; with residual */
    void *y;                 /* out [tokens, hidden]; NULL where q is enough */
    float *mean;             /* out [tokens], or NULL */
    float *rstd;             /* out [tokens], or NULL */
    int8_t *q;               /* out [tokens, hidden], or NULL */
    float *q_scales;         /* out [tokens], with q */
} gg_norm_problem;

int gg_prepare_norm(gg_handle *h, const gg_norm_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Gradients of the layer norm, from what its run wrote: with c = (x - mean) * rstd and d = dy * gamma,
 *
 *   dx = rstd * (d - mean of d - c * mean of d c) + dsum       dgamma = sum over t of dy c       dbeta = sum over t of dy
 *
 * x is the norm's input: sum where there was a residual, whose gradient is dx, too. dsum is the gradient that reaches the
 * sum by its other way (past the layer), or NULL. dgamma and dbeta are fp32, either may be NULL; the same inputs give the same bits. dx may be
 * the same array as dy or dsum. A row whose squares pass fp32 (rstd 0) has dx = dsum and adds nothing to dgamma. Limits as gg_prepare_norm's. */
typedef struct gg_norm_grad_problem {
    int32_t dtype;
    int32_t param_type;      /* of gamma */
    int64_t tokens;
    int64_t hidden;
    const void *x;           /* [tokens, hidden] */
    const float *mean;       /* [tokens] */
    const float *rstd;       /* [tokens] */
    const void *gamma;       /* [hidden], or NULL = 1 */
    const void *dy;          /* [tokens, hidden] */
    const void *dsum;        /* [tokens, hidden] or NULL */
    void *dx;                /* out [tokens, hidden] */
    float *dgamma;           /* out [hidden], or NULL */
    float *dbeta;            /* out [hidden], or NULL */
} gg_norm_grad_problem;

int gg_prepare_norm_grad(gg_handle *h, const gg_norm_grad_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Rows rounded to 8-bit integers with a scale each:
 *
 *   scales_r = max_k |x_rk| / 127 (fp32)      q_rk = the whole number nearest to 127 x_rk / max_k |x_rk|, halves to the even one
 *
 * of the exact quotient. A row of zeros has scale 0; one that holds NaN or an infinity has scale NaN and q 0, so that what is made of it
 * is NaN. The weights of gg_prepare_i8 are made so from [experts * n, k]. k a multiple of 8; x and q 16-byte aligned. */
typedef struct gg_quant_problem {
    int32_t dtype;           /* bf16, fp16 or fp32 */
    int64_t rows;
    int64_t k;
    const void *x;           /* [rows, k] */
    int8_t *q;               /* out [rows, k] */
    float *scales;           /* out [rows] */
} gg_quant_problem;

int gg_prepare_quant(gg_handle *h, const gg_quant_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Products with 8-bit weights, for any number of rows an expert (decoding and prompts):
 *
 *   out[r, n] = x_scales[row(r)] * scales[e, n] * sum_k x[row(r), k] weight[e, n, k]
 *
 * for the rows r of expert e, offsets[e] <= r < offsets[e + 1]; row(r), offsets, src and the rows of no expert as in gg_prepare_w4. x is
 * [.., k] in 8 bits with x_scales, or, where x_scales is NULL, in dtype: then the run rounds its rows first as gg_prepare_quant does (into
 * the handle's memory). The sum is exact in 32 bits; its value is rounded to fp32 and multiplied by the scales there, and the result rounded
 * once to dtype. A row whose src is no slot is zero (or NaN, with a scale that is not finite) and reported. A scale that is not finite makes
 * NaN or infinities of its row or column alone.
 *
 * dtype bf16 or fp16; experts 1..1024, n a multiple of 8, k a multiple of 16 up to 131056; x, weight and out 16-byte aligned. */
typedef struct gg_i8_problem {
    int32_t dtype;           /* of out, and of x without x_scales */
    int32_t experts;
    int32_t top_k;           /* with src */
    int64_t n;
    int64_t k;
    int64_t rows;            /* rows of out */
    int64_t tokens;          /* rows of x, with src */
    const void *x;           /* [tokens, k] with src, else [rows, k] */
    const float *x_scales;   /* [tokens or rows], or NULL: x is in dtype */
    const int8_t *weight;    /* [experts, n, k] */
    const float *scales;     /* [experts, n] */
    const int32_t *offsets;  /* [experts + 1] */
    const int32_t *src;      /* [rows] or NULL */
    void *out;               /* [rows, n] */
} gg_i8_problem;

int gg_prepare_i8(gg_handle *h, const gg_i8_problem *p, gg_stream_t stream, char *why, size_t why_len);

/* Backend::run() (common/backend.hpp:67; ck_kernel/ck_grouped_gemm.cpp:140, :114-121). Timed:
 * enqueues one grouped GEMM on `stream` and does not synchronise: one kernel launch, or two for
 * a split launch ("tail_launch" below). After one of the layer operators' prepare calls it enqueues
 * that operator instead. */
int gg_run(gg_handle *h, gg_stream_t stream);

/* Backend::release() (common/backend.hpp:69; ck_kernel/ck_grouped_gemm.cpp:142-146): frees
 * what gg_prepare() allocated. The handle can be prepared again. */
void gg_release(gg_handle *h);

/* Backend::detail() (common/backend.hpp:71; ck_kernel/ck_grouped_gemm.cpp:216): kernel variant,
 * tile shape, stages and grid of the prepared problem. Valid until the next prepare/release. */
const char *gg_detail(const gg_handle *h);

/* Message of the last failed call on this handle ("" if none). */
const char *gg_last_error(const gg_handle *h);

/* Synchronises `stream`, then reads and clears the kernel's device status word: 0 when every
 * launch since the last read finished normally, otherwise the first bounded-wait timeout code
 * (0x1000 | role << 8 | barrier) or, in the bounds-checked debug build, the first failed check
 * (0x2000 | site: 1 tile decode, 2 direct store, 3 TMA store box, 4 split-K workspace,
 * 5 arrival counter; the checked access was skipped). The outputs of every launch since the last read are then
 * unreliable (an aborted launch stops part-way and can leave the dynamic-dispatch tile counter
 * and split-K arrival counts behind; this call resets them, so later launches are sound again).
 * No counterpart in the reference, whose kernel cannot time out (its only device-side guard is
 * a trap, ck_kernel/fast_epilogue.hpp:38-41). */
int gg_device_status(gg_handle *h, gg_stream_t stream, uint32_t *status);

/* Override the automatic choices of gg_prepare / gg_prepare_grad (takes effect at the next
 * prepare):
 *   "variant"    -1 auto, 0 = 2-CTA 256x256 tile, 1 = 1-CTA 128x256, 2 = 1-CTA 128x128
 *   "band"       tiles per raster band (default chosen per shape), 0 = auto
 *   "raster"     -1 auto (= 0), 0 = bands of M tiles (weight panels shared), 1 = bands of N tiles
 *   "bn"         tile width (multiple of 16, <= the variant's), 0 = auto (cost model)
 *   "split"      K splits per split tile (split-K with an fp32 workspace), 0 = auto, 1 = none
 *   "split_tail" -1 auto, 0 = split every tile, 1 = split only the tiles of what would be a
 *                partial last wave (their units run first, whole tiles after them)
 *   "stream_k"   0 (default) = off, -1 = the cost model decides, 1 = stream-K over the tiles of
 *                what would be a partial last wave, 2 = over those and one full wave more: their
 *                K atoms are dealt out in equal contiguous ranges to all CTAs (pairs), tiles cut
 *                at arbitrary atoms are summed through an fp32 workspace (forward and dgrad;
 *                refused with "split" > 1, for wgrad, and where the tiling has no partial wave)
 *   "store"      -1 auto (direct stores from registers for tiles with >= 16 K atoms, staging +
 *                TMA stores for shorter ones), 0 = always TMA stores, 1 = always direct stores
 *   "sched"      0 (default) = static round-robin (cluster c runs tiles c, c + C, ...), 1 = dynamic
 *                dispatch: a cluster takes its next tile from a counter in the handle's device
 *                memory as it finishes one, so tiles that share a weight panel stay in step all
 *                launch long (fewer DRAM re-reads, but measured slower at the power cap), -1 =
 *                dynamic for launches of whole tiles with more tiles than CTAs / pairs. The counter
 *                is zero between launches, so launches of one handle must not overlap on the GPU
 *                (order them on one stream, as for any handle)
 *   "l2_a", "l2_b" forward op: L2 eviction priority of the A operand's (x) and the B operand's
 *                (weights) TMA loads: 0 no hint, 1 evict_first, 2 evict_last; l2_a -1
 *                (its default) = evict_last where the launch's weights outweigh its activations at
 *                least 4 : 1 and it runs at least 64 waves of tiles (many experts with few tokens
 *                each: over a long launch the streaming weights would push out activation rows
 *                that later tiles of the expert still read), no hint otherwise; l2_b defaults to 0.
 *                Results are unchanged by either. Backward operations ignore both (in the dgrad
 *                producer the hinted load form measured slower than any hint saved)
 *   "tail_launch" -1 auto (default), 0 off, 1 on: with the 2-CTA variant (forward and dgrad, no
 *                split-K or stream-K), the rows of each group's last 256-row tile, where they are at
 *                most 128, go to a second launch of the one-CTA kernel (128-row tiles) right behind
 *                the first in the stream; gg_run then enqueues two kernels. Automatic when at least
 *                5% of the pair m-tiles are such remainders (skewed routing: many small experts)
 *   "half_tiles" 0 off (default), 1 / -1 on: with the 2-CTA variant (forward and dgrad, no
 *                split-K or stream-K, a tile width that is a multiple of 32), a group whose last
 *                256-row tile holds at most 128 rows runs that tile half height (an M = 128 pair
 *                MMA, 64 rows per CTA). Measured slower than the split launch and than padding on
 *                B200 (a half tile costs ~0.9 of a whole one), so it is off unless asked for
 *   "tile_order" whole tiles (no split-K), and for forward / dgrad one launch (no split launch):
 *                0 group order (default), 1 interleaved, -1 interleaved when each kind below holds
 *                at least 5% of the launch's cost. With interleaving, gg_prepare plans the launch's
 *                tile order on the host: tiles of two kinds are merged so that both are dealt out
 *                at the same fraction of their total cost, and the list is copied to the handle's
 *                device memory; "sched" still picks static or dynamic dispatch over it. The kinds:
 *                wgrad, groups with a short reduction (few rows, bound by their output stores) and
 *                groups with a long one (bound by the tensor cores); forward / dgrad, groups with
 *                few m-tiles (bound by reading their weight panels from DRAM) and groups with many.
 *                Measured on B200 under skewed routing (256 experts): wgrad slower than group order
 *                (707 static / 764 dynamic vs 815 TFLOPS); forward with half tiles and dynamic
 *                dispatch level with the split launch at the power cap (1034 vs 1059 TFLOPS), so
 *                it is off unless asked for
 *   "pdl"        1 (default) = launch with programmatic stream serialisation, so the launch and
 *                on-chip set-up overlap the previous kernel in the stream; 0 = plain launch
 *   "max_ctas"   cap on the persistent grid (0 = one CTA per SM)
 *   "timeout_ms" bounded-wait limit inside the kernel (default 2000)
 *   "test_bounds" test only: 1 = the kernel is told the output has one row fewer than it has, so
 *                the bounds-checked debug build (lib/libgg_b200_debug.so, -DGG_DEBUG) finds the last
 *                row's stores out of bounds, skips them and reports 0x2002 in the status word (the
 *                release build has no checks and stores every row); used to test the checks
 *   "test_stall" test only: 1 = the kernel never loads the first stage of its first CTA (pair),
 *                so that wait runs out after timeout_ms and gg_device_status() reports it (the norm, its
 *                gradients and the 8-bit products: that stage's barrier waits for an arrival that never
 *                comes); used to test failure detection without faulting the GPU
 * Returns GG_OK or GG_ERR_ARG for an unknown key. The knobs are the analogue of the compile-time
 * CkTileConfig (ck_kernel/ck_grouped_gemm_config.hpp:26-86) that the reference edits to tune. */
int gg_set_option(gg_handle *h, const char *key, int64_t value);

/* Destroy the handle (calls gg_release first). */
void gg_destroy(gg_handle *h);

/* Expert-parallel shard of `group_num` groups over `world` GPUs: contiguous ranges, the first
 * (group_num % world) ranks get one extra group. Writes [*g0, *g1) for `rank`. Pure host
 * arithmetic (no CUDA). The reference has no multi-GPU path; its only split of experts is the
 * shape generator's EP divisor (scripts/gen_shapes.py:43-48). Returns GG_ERR_ARG on bad input. */
int gg_expert_shard(int32_t group_num, int32_t world, int32_t rank, int32_t *g0, int32_t *g1);

/* Library ABI version (incremented on incompatible change). */
int gg_abi_version(void);

/* One grouped GEMM with no allocation at all: the same computation and result as
 * gg_prepare() + gg_run(), for callers that cannot allocate device memory when they call, e.g. an
 * engine that has reserved the GPU's memory for its own pool, a plugin host with a fixed memory
 * budget, or a latency-critical path that must not call cudaMalloc/cudaFree (they can
 * synchronise the device). No counterpart in the reference, whose backend allocates its
 * argument buffer in prepare (ck_kernel/ck_grouped_gemm.cpp:209).
 *
 * The per-group tile/row offsets and the kernel's status word live in one fixed device array
 * inside the library (about 8 KB, held by every GPU that loads the library until the process
 * exits), so group_num is limited to 1024; larger problems are refused with GG_NOT_SUPPORTED and
 * a reason in `why`. Nothing is allocated, neither device memory nor host heap memory.
 * Enqueues two kernels on `stream` (one writes the call's group offsets into the array, passed
 * by value as its launch parameter; then the grouped GEMM) and returns without waiting for the
 * GPU, unless `status_out` is non-NULL: then it waits for the stream and stores the status word
 * there (0 = every bounded wait finished; GG_ERR_DEVICE is returned otherwise).
 *
 * The status word is shared by every call on the device and is sticky: a bounded-wait timeout
 * in any call stays recorded (and makes the waits of later calls give up early, leaving their
 * output incomplete) until a call with a non-NULL `status_out` reports it and clears it. A call
 * with `status_out == NULL` therefore reports nothing itself; a caller that never passes
 * `status_out` cannot detect a timeout.
 *
 * The first call on each device does a one-time set-up (it looks up the array's device address
 * and the kernels' launch limits); make that first call before any stream capture. Every call
 * on a device shares the one array and each call overwrites it, so calls whose kernels may
 * overlap on the GPU (different streams without ordering between them) race; calls in order on
 * one stream do not. Errors are reported in `why` (there is no handle for gg_last_error). */
int gg_run_noalloc(const gg_problem *p, gg_stream_t stream, uint32_t *status_out, char *why, size_t why_len);

#ifdef __cplusplus
}
#endif

#endif /* GG_B200_H */
