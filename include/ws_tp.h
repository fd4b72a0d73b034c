/*
 * ws_tp.h -- C ABI of the B200 (sm_100a) tensor-parallel reduction library.
 *
 * One `ws_tp_t` is one rank's endpoint of a tensor-parallel group of 1, 2, 4 or 8
 * ranks on one NVLink/NVSwitch node.  The fused operators below run the
 * row-parallel block-scaled GEMM of a reduction point and the fp32 exchange that
 * follows it in ONE kernel: partial sums are stored straight into every peer's
 * memory and summed in rank order 0,1,..,R-1, so every rank ends with identical
 * bits.  They replace, in msuiche/weightstream, the GEMM launches of
 * `crates/weightstream-gpu/src/engine.rs` together with the host-side
 * `trait Collectives` (`engine.rs:287-294`) that `crates/weightstream-transport`
 * implements over RoCE (`src/ring.rs:395-437`).
 *
 * Conventions
 *  - every function returns a `ws_status_t` (0 = ok, negative = error); nothing
 *    aborts the process or throws.  `ws_tp_last_error` gives the text.
 *  - all device work is enqueued on the caller's stream (`void*` = cudaStream_t);
 *    the device-resident entry points never synchronise.  A peer that does not
 *    arrive within `wait_ms` makes the kernel record WS_ERR_TIMEOUT in a status
 *    word and return (fail-stop, as `ring.rs:439-458`); `ws_tp_check` reads it.
 *  - ranks are lock-step SPMD: every rank issues the same sequence of fused
 *    operators / collectives on its endpoint (`ring.rs:334-337`).
 *  - per-rank slicing keeps the reference's contract `rank*len/world`
 *    (`engine.rs:1477-1480` K slices, `:1194-1195` experts, `:3107-3108` vocab).
 */
#ifndef WS_TP_H
#define WS_TP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WS_MAX_WORLD 8
#define WS_IPC_HANDLE_BYTES 128

typedef int32_t ws_status_t;
enum {
    WS_OK = 0,
    WS_ERR_INVALID = -1,      /* bad argument: shape, alignment, shard bounds   */
    WS_ERR_CUDA = -2,         /* a CUDA runtime / driver call failed             */
    WS_ERR_TIMEOUT = -3,      /* a peer's partial did not arrive within wait_ms  */
    WS_ERR_SEQUENCE = -4,     /* ranks disagree on the step count (host check, or a peer's
                                 partial tagged with a later step: ring.rs:488-499)          */
    WS_ERR_CAPACITY = -5,     /* the step exceeds what the endpoint was sized for */
    WS_ERR_UNSUPPORTED = -6
};

enum { WS_SCALE_UE8M0 = 0, WS_SCALE_F32 = 1 };   /* weight-scale element type */
enum { WS_ACT_BF16 = 0, WS_ACT_F32 = 1 };        /* activation element type   */

typedef struct ws_tp ws_tp_t;

typedef struct {
    int32_t max_m;          /* most activation rows (tokens) in one fused step           */
    int32_t max_n;          /* widest reduced output row (model dim)                     */
    int32_t max_vocab;      /* full vocabulary for the lm_head gather (0 = not used)     */
    int32_t wait_ms;        /* bound on every wait for a peer; <= 0 selects 2000 ms      */
    int32_t num_ctas;       /* persistent CTAs per rank; 0 = one per SM                  */
    int32_t reserved[3];
} ws_tp_config_t;

typedef struct { uint8_t bytes[WS_IPC_HANDLE_BYTES]; } ws_ipc_handle_t;

/* ---- endpoint life cycle: replaces tp4::join + Ring::new
 *      (crates/weightstream-gpu/src/tp4.rs:191-312, crates/weightstream-transport/src/ring.rs:115-217) */
ws_status_t ws_tp_create(int32_t world, int32_t rank, int32_t device,
                         const ws_tp_config_t *cfg, ws_tp_t **out);
ws_status_t ws_tp_destroy(ws_tp_t *tp);
/* One process per rank: export this rank's exchange memory, then hand every
 * rank's handle (index = rank) to ws_tp_connect_ipc.  The caller moves the
 * bytes between processes (the reference does the same over its TCP control
 * plane, crates/weightstream-transport/src/ctrl.rs:12-29). */
ws_status_t ws_tp_export_handle(ws_tp_t *tp, ws_ipc_handle_t *out);
ws_status_t ws_tp_connect_ipc(ws_tp_t *tp, const ws_ipc_handle_t *handles, int32_t n);
/* The same exchange without a host framework: the ranks trade their handles over TCP (rank 0 listens on
 * host:port, the others connect, retrying until timeout_ms has passed) and every rank connects as by
 * ws_tp_connect_ipc.  Replaces, for this purpose, the reference's TCP control plane
 * (crates/weightstream-transport/src/ctrl.rs:12-29, group bring-up in
 * crates/weightstream-gpu/src/tp4.rs:191-312).  WS_ERR_TIMEOUT when a rank does not show up,
 * WS_ERR_INVALID when a rank reports another world size, a rank number twice or one out of range. */
ws_status_t ws_tp_connect_tcp(ws_tp_t *tp, int32_t rank, int32_t world, const char *host, int32_t port, int32_t timeout_ms);
/* The rendezvous by itself (no device involved): every rank contributes `len` bytes and receives all
 * ranks' bytes in rank order in `out` (world * len bytes). */
ws_status_t ws_tcp_allgather(int32_t rank, int32_t world, const char *host, int32_t port, const void *in, void *out,
                             int32_t len, int32_t timeout_ms);
/* One process driving all ranks (several devices with peer access, or several
 * virtual ranks on one device for single-GPU testing). */
ws_status_t ws_tp_connect_local(ws_tp_t *const *ranks, int32_t n);

/* Synchronise `stream`, then report the status word the kernels wrote. */
ws_status_t ws_tp_check(ws_tp_t *tp, void *stream);
/* Replaces Collectives::stats (engine.rs:291-293). */
const char *ws_tp_last_error(ws_tp_t *tp);
ws_status_t ws_tp_stats(ws_tp_t *tp, uint64_t *steps, uint64_t *launches);
int32_t ws_tp_num_ctas(ws_tp_t *tp);

/* ---- FP8 row-parallel GEMM + all-reduce -------------------------------------------------
 * Replaces emit8 + gemm_q8(wo_b) + Collectives::allreduce at the attention output
 * projection (engine.rs:3988-4029; batched form :6158-6181) and the same triple
 * for a K-sharded shared-expert down projection (reference CPU form
 * crates/weightstream-ref/src/moe.rs:245-249).
 *
 * out[m, n] = sum over ranks r (in rank order) of
 *             sum_k fp8_act(x_r)[m, k] * e4m3(w_r[n, k]) * scale_r(n, k)
 * where fp8_act is the reference's dynamic per-32 activation quantisation
 * (crates/weightstream-ref/src/actquant.rs:21-57) applied in the kernel prologue, and
 * scale_r(n, k) = scales[((row0 + n) / block_n) * scale_ld + (k0 + k) / block_k]. */
typedef struct {
    const void *x;            /* [m, k] activations of this rank's K slice, row stride ldx (elements) */
    int64_t ldx;
    int32_t x_dtype;          /* WS_ACT_BF16 or WS_ACT_F32                                            */
    int32_t m, n, k;          /* k = this rank's slice length (multiple of 32)                        */
    const uint8_t *w;         /* E4M3 bytes [n, k], row stride ldw bytes (multiple of 16)             */
    int64_t ldw;
    const void *scales;       /* scale matrix this rank holds                                         */
    int64_t scale_ld;         /* elements per scale row                                               */
    int32_t scale_kind;       /* WS_SCALE_UE8M0 (reference: 32x32) or WS_SCALE_F32 (128x128)          */
    int32_t block_n, block_k; /* scale block shape; powers of two, block_n >= 16, block_k >= 32       */
    int64_t row0, k0;         /* offset of w[0,0] inside the held scale matrix (row0 multiple of 16)  */
    float *out;               /* [m, n] fp32, row stride n                                            */
} ws_fp8_gemm_args_t;

ws_status_t ws_fp8_rowpar_gemm_allreduce(ws_tp_t *tp, const ws_fp8_gemm_args_t *args, void *stream);
/* Same step for n endpoints held by one process (args[i] and streams[i] belong to ranks[i]). */
ws_status_t ws_fp8_rowpar_gemm_allreduce_group(ws_tp_t *const *ranks, int32_t n,
                                               const ws_fp8_gemm_args_t *args, void *const *streams);

/* ---- MoE routed-expert down projection + combine + all-reduce ---------------------------
 * Replaces emit8 + moe_grouped_tl(Down) + moe_combine_f32 + Collectives::allreduce
 * (engine.rs:4207-4239, :4513-4522; reference CPU form moe.rs:75-84, :150, :203-207).
 * For token t: out[t] = sum over ranks of the sum, in ascending expert id, over the
 * routes of t whose expert is local, of fp4_gemv(W2[e], fp8_act(h[route] * weight[route])).
 * The routing weight multiplies the hidden BEFORE quantisation (moe.rs:99-102). */
typedef struct {
    const void *h;            /* [m*top_k, k] hidden of every route (row = t*top_k + slot)    */
    int64_t ldh;
    int32_t h_dtype;
    int32_t m, n, k, top_k;
    const int32_t *route_ids; /* device [m, top_k] global expert ids, -1 = empty slot         */
    const float *route_w;     /* device [m, top_k]                                            */
    const uint8_t *w2;        /* local slab [e_len][n][k/2] packed E2M1, low nibble = even K  */
    const uint8_t *s2;        /* [e_len][n][k/32] UE8M0                                       */
    int32_t e_start, e_len;   /* this rank owns experts [e_start, e_start+e_len)              */
    float *out;               /* [m, n] fp32                                                  */
} ws_moe_down_args_t;

ws_status_t ws_moe_down_combine_allreduce(ws_tp_t *tp, const ws_moe_down_args_t *args, void *stream);
ws_status_t ws_moe_down_combine_allreduce_group(ws_tp_t *const *ranks, int32_t n,
                                                const ws_moe_down_args_t *args, void *const *streams);

/* ---- vocab-sharded lm_head + all-gather + argmax ------------------------------------------
 * Replaces bf16_gemv(head) + Collectives::allgather + argmax_rows
 * (engine.rs:2647-2667, :2687-2703; tie rule crates/weightstream-ref/src/sample.rs:13-23:
 * the lowest index among equal maxima wins, all -inf gives 0).
 * `g` describes this rank's vocab shard (g.n = local rows, g.out unused);
 * `vocab_row0` is the shard's first global row and `vocab` the full size. */
typedef struct {
    ws_fp8_gemm_args_t g;
    int64_t vocab_row0;
    int32_t vocab;
    int32_t reserved;
    float *logits;            /* [m, vocab] fp32 or NULL when only the argmax is wanted */
    uint32_t *argmax;         /* [m] or NULL                                            */
} ws_lm_head_args_t;

ws_status_t ws_lm_head_allgather_argmax(ws_tp_t *tp, const ws_lm_head_args_t *args, void *stream);
ws_status_t ws_lm_head_allgather_argmax_group(ws_tp_t *const *ranks, int32_t n,
                                              const ws_lm_head_args_t *args, void *const *streams);

/* ---- bare collectives on device buffers: Collectives::allreduce / ::allgather
 *      (engine.rs:287-290, ring.rs:395-437) without the host round trip ------------------- */
ws_status_t ws_allreduce_f32(ws_tp_t *tp, const float *in, float *out, int64_t len, void *stream);
ws_status_t ws_allgather_f32(ws_tp_t *tp, const float *in, float *out, int64_t len, void *stream);
ws_status_t ws_allreduce_f32_group(ws_tp_t *const *ranks, int32_t n, const float *const *in,
                                   float *const *out, int64_t len, void *const *streams);
ws_status_t ws_allgather_f32_group(ws_tp_t *const *ranks, int32_t n, const float *const *in,
                                   float *const *out, int64_t len, void *const *streams);

/* ---- host-buffer forms: the exact shape of the reference trait (host slice in, host
 *      result out, error = abort the decode).  They copy, launch, synchronise and check. --- */
ws_status_t ws_allreduce_f32_host(ws_tp_t *tp, const float *in, float *out, int64_t len);
ws_status_t ws_allgather_f32_host(ws_tp_t *tp, const float *in, float *out, int64_t len);
ws_status_t ws_fp8_rowpar_gemm_allreduce_host(ws_tp_t *tp, const ws_fp8_gemm_args_t *dev_weights,
                                              const void *x_host, float *out_host);

/* ---- activation quantisation alone: act_quant_fp8_emit
 *      (crates/weightstream-cuda/kernels/actquant.cu:47-83), bit-exact with
 *      crates/weightstream-ref/src/actquant.rs:21-57.  q [m, k] E4M3, sexp [m, k/32] UE8M0. */
ws_status_t ws_act_quant_fp8(const void *x, int64_t ldx, int32_t x_dtype, int32_t m, int32_t k,
                             uint8_t *q, uint8_t *sexp, void *stream);

/* Scheduling knob with no counterpart in the reference: 1 (default) deals the output rows
 * that do not fill whole 16-row tiles on every CTA out row by row, so that every SM streams
 * the same number of bytes; 0 hands each leftover tile to one CTA whole. */
ws_status_t ws_tp_set_split(ws_tp_t *tp, int32_t on);
/* Kernel choice, also without counterpart in the reference.  0 (default) automatic: FP8 steps run
 * one or two activation rows on CUDA cores and three or more (two rows of shards from 24 MB, with
 * UE8M0 scales from 8 MB; one row from 128 MB, lm_head from 32 MB) on the block-scaled tcgen05 kernel;
 * the MoE step runs on its tcgen05 kernel when the shape fits it (k a multiple of 256 and at most 4096,
 * one rank per launch), else on its CUDA-core decode form.  1: the mma.sync
 * formulations.  2: the tcgen05 kernels wherever the shape fits.  3: the CUDA-core kernels (MoE: the
 * decode form).  All choices give results within the same tolerance of the reference arithmetic;
 * ranks of one group must make the same choice. */
ws_status_t ws_tp_set_kernel(ws_tp_t *tp, int32_t which);

/* ---- FP8 GEMM for callers that must not allocate ------------------------------------------
 * No counterpart in the reference.  Some hosts embed this library where device memory may
 * not be allocated on their behalf: a runtime that hands out one fixed arena at start-up and
 * forbids cudaMalloc afterwards, code running inside a memory-pool or capture-style region
 * where an allocation is an error, or a plug-in that has no endpoint (ws_tp_create allocates
 * the exchange region).  This is the single-rank form of ws_fp8_rowpar_gemm_allreduce (same
 * arguments, same kernel, out = the whole sum since there is one rank) whose scratch -- the
 * kernel's status word, step counter and arrival counters -- is a fixed array inside
 * the library image (WS_STATIC_SCRATCH_BYTES per GPU that loads the library, held until the
 * process exits).  It calls no cudaMalloc / cudaFree and no allocating library routine.
 *
 *  - limits: m <= WS_STATIC_MAX_M and n <= WS_STATIC_MAX_N; beyond them WS_ERR_CAPACITY with a
 *    message in `err` (optional buffer of err_len bytes).
 *  - the first call on a device looks the array's device address up and raises the kernel's
 *    shared-memory limit; make that first call before any stream capture begins.
 *  - all calls on a device share the one array, which keeps the previous call's contents; the
 *    entry point clears the counters and the status word on `stream` before the kernel.  Two
 *    calls that overlap on the GPU (different streams, no ordering) race on it.
 *  - both functions make `device` the calling thread's current device and leave it so.
 *  - the launch is asynchronous and returns WS_OK once enqueued.  A bounded wait inside the kernel
 *    that gives up (a weight tile that never lands) is recorded in the array's status word, which
 *    the next call clears: call ws_fp8_gemm_static_scratch_check after the launch -- it
 *    synchronises `stream`, reads the word (4 bytes, no allocation) and returns WS_OK or the
 *    recorded error with its text in `err` -- before trusting `out`. */
#define WS_STATIC_MAX_M 8
#define WS_STATIC_MAX_N 1048576
#define WS_STATIC_SCRATCH_BYTES 1024
ws_status_t ws_fp8_gemm_static_scratch(const ws_fp8_gemm_args_t *args, int32_t device, void *stream,
                                       char *err, size_t err_len);
ws_status_t ws_fp8_gemm_static_scratch_check(int32_t device, void *stream, char *err, size_t err_len);

/* ---- operators between the steps --------------------------------------------------------------
 * What an engine does between two reduction points, on the tensors that the steps above take and
 * return.  They need no endpoint and run on the calling thread's current device.  Types are
 * WS_ACT_BF16 or WS_ACT_F32, sums and statistics are held in 32 bits.  Every tensor, results among them,
 * is aligned to its type, and widths stay below 2^31 - 4096 (the vocabulary below 2^31 - 65536); else
 * WS_ERR_INVALID.  `err` (optional, err_len bytes) gets the text of an error.  m = 0 launches nothing. */

/* Norms before and after a block with its gate, residual scale and the residual stream:
 *   u = y, or with post_weight  y * rsqrt(mean(y^2) + eps) * (weight_offset + post_weight)
 *   hidden = residual_scale * residual + block_scale * act(gate) * u
 *   normed = hidden * rsqrt(mean(hidden^2) + eps) * (weight_offset + next_weight), from the unrounded hidden
 * (takes the place of the reference's `rmsnorm` launches between its blocks). */
enum { WS_GATE_LINEAR = 0, WS_GATE_SIGMOID = 1 };
typedef struct {
    const void *y;            /* [m, n] the block's output, row stride ldy (elements, as all strides)   */
    int64_t ldy;
    const void *residual;     /* [m, n] or NULL (no residual)                                           */
    int64_t ldr;
    const void *gate;         /* NULL: 1.  gate[row * ldg + i * gate_inc]: ldg 0 shares one row of gates, */
    int64_t ldg;              /*   gate_inc 0 is one gate a row, 1 one a value                          */
    const void *post_weight;  /* [n] or NULL: no norm of the block's output                             */
    const void *next_weight;  /* [n]; needed with normed                                                */
    void *hidden;             /* [m, n] or NULL; may be `residual` itself                               */
    int64_t ldh;
    void *normed;             /* [m, n] or NULL                                                         */
    int64_t ldn;
    int32_t m, n, gate_inc, gate_act;
    int32_t y_dtype, residual_dtype, gate_dtype, weight_dtype, hidden_dtype, normed_dtype;
    float weight_offset, eps, residual_scale, block_scale;
} ws_block_norm_args_t;
ws_status_t ws_block_norm(const ws_block_norm_args_t *args, void *stream, char *err, size_t err_len);

/* Scores of one given token a row on the vocabulary head's logits:
 *   lse = log sum exp(logits);  logprob = logits[token] - lse;  entropy = lse - sum softmax(logits) * logits
 *   rank = how many entries come before the token, larger ones first and equal ones by index (0: it is the argmax)
 *   top_id, top_logprob: the `top` entries that come first; masked (-inf) and NaN logits are never among them,
 *   places that stay empty hold -1 and -inf.
 * A token outside [0, vocab) is none: logprob 0, rank -1.  A row that is masked whole has logprob -inf, entropy 0.
 * NaN or +inf in a row make its logprob, entropy and top_logprob NaN; a token whose own logit is NaN has rank -1.
 * Order of the entries as in argmax (crates/weightstream-ref/src/sample.rs:13-23). */
#define WS_MAX_TOP 32
typedef struct {
    const void *logits;       /* [m, vocab], row stride ld (elements)   */
    int64_t ld;
    const void *tokens;       /* [m] int32 or int64 (token_bytes 4 or 8) */
    float *logprob;           /* [m]                                     */
    float *entropy;           /* [m]                                     */
    int32_t *rank;            /* [m]                                     */
    int32_t *top_id;          /* [m, top], NULL with top = 0             */
    float *top_logprob;       /* [m, top], NULL with top = 0             */
    int32_t m, vocab, top, dtype, token_bytes, reserved;
} ws_token_logprobs_args_t;
ws_status_t ws_token_logprobs(const ws_token_logprobs_args_t *args, void *stream, char *err, size_t err_len);

/* Low-rank adapters of many requests beside a shared projection:
 *   out[t] = y[t] + scale[ids[t]] * b[ids[t]] (a[ids[t]] x[t])
 * Tokens with an id outside [0, adapters), such as -1, have no adapter: out = y, shrunk rows are zeros.
 * ws_lora_add is the whole; where the projection is sharded over K every rank calls ws_lora_shrink on its slice of x
 * and of a, the ranks add the shrunk rows up (ws_allreduce_f32) and each calls ws_lora_expand.
 * The adapters are bf16 (an infinite weight makes its results infinite or NaN), the products' sums and
 * the shrunk rows fp32.  Up to 512 tokens need no workspace; more take
 * ws_lora_workspace(m, adapters, rank) bytes (16-byte aligned) that the call writes first, so calls on one stream may share
 * it, and at most 16384 adapters (WS_ERR_CAPACITY beyond). */
#define WS_LORA_MAX_RANK 128
typedef struct {
    const void *x;            /* [m, k] activations, row stride ldx                 (add, shrink) */
    int64_t ldx;
    const void *y;            /* [m, n] the projection's result, row stride ldy     (add, expand) */
    int64_t ldy;
    void *out;                /* [m, n] of y's type, row stride ldo; may be y itself (add, expand) */
    int64_t ldo;
    const void *a;            /* [adapters, rank, k] bf16                            (add, shrink) */
    const void *b;            /* [adapters, n, rank] bf16                            (add, expand) */
    const int32_t *ids;       /* [m]                                                 (all)         */
    const float *scale;       /* [adapters], or NULL: 1                              (add, expand) */
    float *shrunk;            /* [m, rank] fp32          (shrink writes it, expand reads it)       */
    void *workspace;
    int64_t workspace_bytes;
    int32_t m, k, n, rank, adapters, x_dtype, y_dtype, reserved;
} ws_lora_args_t;
int64_t ws_lora_workspace(int32_t m, int32_t adapters, int32_t rank);
ws_status_t ws_lora_add(const ws_lora_args_t *args, void *stream, char *err, size_t err_len);
ws_status_t ws_lora_shrink(const ws_lora_args_t *args, void *stream, char *err, size_t err_len);
ws_status_t ws_lora_expand(const ws_lora_args_t *args, void *stream, char *err, size_t err_len);

/* Norms of queries and keys, head by head, and the rotation of positions:
 *   u = x * rsqrt(mean(x^2) + eps) * (weight_offset + weight)      over a head's d values (norm = 0: x * (weight_offset + weight))
 *   a' = scale (a cos - b sin), b' = scale (a sin + b cos)         angle = position * inv_freq[i], for the pairs
 *   (a, b) = (u[start + i], u[start + pairs + i]), or with interleaved (u[start + 2 i], u[start + 2 i + 1]);
 * the other values of u stay.  The angle is exact up to positions of 2^53.  pairs = 0: no rotation (positions and inv_freq unused).
 * q_out and k_out may be q and k themselves.  (Takes the place of the reference's `rmsnorm` and `rope` launches in front of its
 * attention.) */
#define WS_MAX_PAIRS 1024
typedef struct {
    const void *q, *k;        /* [m, heads, d]; k NULL: queries alone                                       */
    int64_t ldqt, ldqh, ldkt, ldkh;       /* strides from token to token and head to head (elements)          */
    void *q_out, *k_out;
    int64_t ldqt_out, ldqh_out, ldkt_out, ldkh_out;
    const void *q_weight, *k_weight;      /* [d] or NULL: 1 (without weight_offset)                           */
    const void *positions;    /* [m] int32 or int64 (position_bytes 4 or 8)                                  */
    const float *inv_freq;    /* [pairs]                                                                     */
    int32_t m, q_heads, k_heads, d, pairs, start, interleaved, norm, dtype, weight_dtype, position_bytes;
    float eps, weight_offset, scale;
} ws_head_norm_rope_args_t;
ws_status_t ws_head_norm_rope(const ws_head_norm_rope_args_t *args, void *stream, char *err, size_t err_len);

/* Experts of every token from the gate's logits, in the form that the routed steps read:
 *   score = softmax(logits), sigmoid(logits) or sqrt(ln(1 + exp(logits)));  key = score + bias (score without one)
 *   ids = the top_k experts by key, larger first and equal ones by index
 *   weights = scale * score, with renormalize divided by the sum of the chosen scores
 * Experts whose logit is -inf or NaN, or whose key is NaN (all of a row's with softmax and a logit of +inf), are never chosen; places
 * that stay empty hold id -1 and weight 0.
 * The order is that of the definition: near ones are compared in 64 bits.  (Takes the place of the reference's `moe_select`.) */
enum { WS_SCORE_SOFTMAX = 0, WS_SCORE_SIGMOID = 1, WS_SCORE_SQRTSOFTPLUS = 2 };
#define WS_ROUTE_MAX_EXPERTS 1024
#define WS_ROUTE_MAX_TOP_K 32
typedef struct {
    const void *logits;       /* [m, experts], row stride ld (elements) */
    int64_t ld;
    const float *bias;        /* [experts] or NULL                       */
    int32_t *ids;             /* [m, top_k]                              */
    float *weights;           /* [m, top_k]                              */
    int32_t m, experts, top_k, score, dtype, renormalize;
    float scale;
} ws_moe_route_args_t;
ws_status_t ws_moe_route(const ws_moe_route_args_t *args, void *stream, char *err, size_t err_len);

/* A whole mixture-of-experts layer of a few tokens over MXFP4 experts, in two kernels and a sum:
 *   g = w1[e] x[t], u = w3[e] x[t];  with limit > 0: g = min(g, limit), u = min(max(u, -limit), limit)
 *   out[t] = sum over t's routes (in the order of their slots) of w2[e] (weight * silu(g) * u)
 * Weights are packed E2M1 (low nibble = even K) with a UE8M0 byte per 32 values of K, as in ws_moe_down_combine_allreduce,
 * every expert's rows one after the other; experts lie w1_stride .. s2_stride bytes apart, so W1 and W3 may be halves of one
 * tensor.  Scale byte 0 counts as 0, 255 gives infinities or NaN, as bytes above 222 (2^95) may: sums are held in fp32 in units of a
 * row's largest activation.  Routes to experts outside [e_start, e_start + e_len), such as
 * -1, are other ranks': out then is this rank's part of the sum (ws_allreduce_f32).
 * act_quant 0: bf16 activations are held as they are, fp32 ones and the weighted hidden in 22 bits or more, both down to 2^-17 of their
 * row's largest (bf16: 2^-29) and below that to 2^-40 of it.  1: x and the weighted hidden are rounded as the fused steps do.
 * Routes and weights may be what the kernel in front of the call on its stream writes; as long as the call runs nothing may
 * change them (the second kernel reads them before the first has ended).
 * hidden and inter are multiples of 32; weights, scales and strides are multiples of 16 bytes.
 * At most 512 routes (m * top_k), 512 local experts, top_k 8 and widths of 24576 (WS_ERR_CAPACITY beyond).  The workspace
 * (ws_moe_layer_workspace bytes, 16-byte aligned) is written first, so calls on one stream may share it. */
typedef struct {
    const void *x;            /* [m, hidden] activations, row stride ldx (elements)  */
    int64_t ldx;
    const int32_t *route_ids; /* [m, top_k] global expert ids                        */
    const float *route_w;     /* [m, top_k]                                          */
    const uint8_t *w1, *s1;   /* [e_len][inter][hidden/2], [e_len][inter][hidden/32] */
    const uint8_t *w3, *s3;   /* as w1 and s1                                        */
    const uint8_t *w2, *s2;   /* [e_len][hidden][inter/2], [e_len][hidden][inter/32] */
    int64_t w1_stride, s1_stride, w3_stride, s3_stride, w2_stride, s2_stride;
    void *out;                /* [m, hidden], row stride ldo                         */
    int64_t ldo;
    void *workspace;
    int64_t workspace_bytes;
    int32_t m, hidden, inter, top_k, e_start, e_len, x_dtype, out_dtype, act_quant;
    float limit;              /* <= 0: none                                          */
} ws_moe_layer_args_t;
int64_t ws_moe_layer_workspace(int32_t m, int32_t top_k, int32_t hidden, int32_t inter);
ws_status_t ws_moe_layer(const ws_moe_layer_args_t *args, void *stream, char *err, size_t err_len);

/* Bias, penalties for repeated tokens and grammar masks on logits, in this order:
 *   z = logits + bias                              (the row's listed tokens; of a token listed twice the last entry counts)
 *   z = z > 0 ? z / repetition : z * repetition    where the token occurs in the row's history
 *   z = z - frequency * count - presence           where count, its occurrences behind the first prompt_lens tokens, is not 0
 *   z = -inf                                       where the row's mask has no bit for the token
 * Row t's history is tokens[offsets[t] .. offsets[t + 1]), its biases likewise; offsets outside [0, n_tokens] are taken to its
 * ends, and tokens outside [0, vocab) ignored.  Bit v % 32 of word v / 32 of a mask allows token v; row t uses mask row
 * mask_rows[t] (NULL: t).  A row whose mask row is outside [0, mask_count), such as -1, has no mask: all its tokens are allowed.  out may
 * be logits itself. */
typedef struct {
    const void *logits;       /* [m, vocab], row stride ld (elements)               */
    int64_t ld;
    void *out;                /* [m, vocab] of the logits' type, row stride ldo      */
    int64_t ldo;
    const int32_t *tokens;    /* [n_tokens] or NULL: no penalties                    */
    const void *offsets;      /* [m + 1] int32 or int64 (offset_bytes 4 or 8)        */
    const int32_t *prompt_lens;                       /* [m] or NULL: 0              */
    const float *repetition, *frequency, *presence;   /* [m] or NULL: 1, 0, 0        */
    const int32_t *bias_ids;  /* [n_bias] or NULL: no biases                         */
    const float *bias;        /* [n_bias]                                            */
    const void *bias_offsets; /* [m + 1] as offsets                                  */
    const uint32_t *mask;     /* [mask_count, ld_mask] words or NULL                 */
    const int32_t *mask_rows; /* [m] or NULL                                         */
    int64_t n_tokens, n_bias, ld_mask;
    int32_t m, vocab, mask_count, offset_bytes, bias_offset_bytes, dtype;
} ws_adjust_logits_args_t;
ws_status_t ws_adjust_logits(const ws_adjust_logits_args_t *args, void *stream, char *err, size_t err_len);

const char *ws_version(void);

#ifdef __cplusplus
}
#endif
#endif
