// C entry points of the operators of a decode step around the reduction points (include/ws_tp.h): norms and rotation of
// heads, routes, a whole expert layer, logits under penalties and masks.  Checks of arguments, choice of kernel, launch.
#include <algorithm>

#include "ws_adjust_kernel.cuh"
#include "ws_heads_kernel.cuh"
#include "ws_layer_kernel.cuh"
#include "ws_ops_host.cuh"
#include "ws_route_kernel.cuh"

using namespace ws;

namespace {

bool aligned_to(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// ---- heads
template <bool F32, bool INTER>
ws_status_t launch_heads(const Err &err, int nu, bool whole, const HeadsParams &p, void *stream) {
    const dim3 grid(p.teams > 1 ? (unsigned)((p.m + p.teams - 1) / p.teams) : (unsigned)p.m * p.groups);
    if (nu == 1) return launch(err, whole ? heads_kernel<F32, INTER, 1, true> : heads_kernel<F32, INTER, 1, false>, grid, kHeadsThreads, 0, 1, stream, p);
    return launch(err, nu == 2 ? heads_kernel<F32, INTER, 2, false> : heads_kernel<F32, INTER, 4, false>, grid, kHeadsThreads, 0, 1, stream, p);
}
template <bool F32>
ws_status_t launch_heads(const Err &err, int nu, bool whole, const HeadsParams &p, void *stream) {
    return p.interleaved ? launch_heads<F32, true>(err, nu, whole, p, stream) : launch_heads<F32, false>(err, nu, whole, p, stream);
}

// ---- routes
// The next of these sizes that holds the experts (4096 tokens of 384 by score and bias 18.8 us with 12 logits a lane, 20.2 with
// 16, 28.9 with 32).
template <bool F32>
ws_status_t launch_route(const Err &err, int n, dim3 grid, void *stream, const RouteParams &p) {
    return launch(err, n <= 2 ? route_kernel<2, F32> : n <= 4 ? route_kernel<4, F32> : n <= 8 ? route_kernel<8, F32> : n <= 12 ? route_kernel<12, F32> : n <= 16 ? route_kernel<16, F32> : route_kernel<32, F32>,
                  grid, kRouteThreads, 0, 1, stream, p);
}

// ---- logits
template <bool F32, bool VEC, int U, int BLOCKS>
ws_status_t launch_adjust(const Err &err, AdjustParams &p, void *stream) {
    constexpr int W = F32 ? 4 : 8, slice = kAdjustThreads * U * W;
    // The places of biases are looked for in the lists, or where these are long have a table of their own.  (A long list in a
    // batch of short ones makes room for one in its blocks.)
    p.bias_table = p.n_bias / p.m > kAdjustFew;
    const int smem = p.tokens || p.bias_ids ? slice * (p.bias_table ? 8 : 4) : 0;
    if (smem > 40 * 1024) {                         // (48 KB with the list)
        const ws_status_t st = allow_smem<adjust_kernel<F32, VEC, U, BLOCKS>>(err, slice * 8);
        if (st != WS_OK) return st;
    }
    const int64_t slices = ((int64_t)p.vocab + (VEC ? W - 1 : 0) + slice - 1) / slice;
    if (slices * p.m > INT32_MAX) return err(WS_ERR_CAPACITY, "%d rows of %d logits: too many for one call", p.m, p.vocab);
    p.slices = (int)slices;
    return launch(err, adjust_kernel<F32, VEC, U, BLOCKS>, dim3((unsigned)(slices * p.m)), kAdjustThreads, (size_t)smem, 1, stream, p);
}
template <bool F32, bool VEC>
ws_status_t launch_adjust(const Err &err, AdjustParams &p, void *stream) {
    // Few rows are cut into more blocks (fp32 rows with 2000 tokens, small and large slices: 1 row 3.9 and 5.1 us, 4 rows 4.7 and
    // 5.5, 9 and 16 rows alike, 32 rows 11.9 and 8.9).
    if ((int64_t)p.m * p.vocab <= 148 * 8192) return launch_adjust<F32, VEC, F32 ? 2 : 1, 6>(err, p, stream);
    return launch_adjust<F32, VEC, F32 ? 8 : 4, F32 ? 4 : 6>(err, p, stream);
}

// ---- layer
constexpr int kLayerSmem = 232448 - (int)sizeof(LayerPlan) - kLayerWarps * 16 * 8 * 4 - 1024;

template <bool FIRST, bool PAIR, bool FULL, int NT, int D>
ws_status_t launch_layer(const Err &err, const LayerParams &p, int smem, void *stream) {
    constexpr auto k = layer_kernel<FIRST, PAIR, FULL, NT, D>;
    const ws_status_t st = allow_smem<k>(err, kLayerSmem);
    return st != WS_OK ? st : launch(err, k, dim3(kLayerBlocks), kLayerThreads, (size_t)smem, 1, stream, p);
}
template <bool FIRST, bool PAIR, bool FULL, int NT>
ws_status_t launch_layer(const Err &err, LayerParams &p, void *stream) {
    const int row = layer_column_pitch(p.k) * (PAIR ? 2 : 1), rest = 2 * kLayerWarps * NT * 4 * 32 * 4;
    auto room = [&](int d) { return (kLayerSmem - rest - kLayerWarps * d * kLayerStage<FULL>) / row; };
    // Routes a pass: as many as the columns hold and the batch can have, less where wide rows leave no room for three stages.
    // Then as many stages as leave room for the rows of a block's passes, of which there are mostly two.
    p.per = std::max(1, std::min({p.m, PAIR ? NT * 4 : 8, room(3)}));
    const int wanted = std::min(p.m * p.top_k, 2 * p.per);
    const int d = room(6) >= wanted ? 6 : room(4) >= wanted ? 4 : 3;
    p.room = std::min(room(d), kLayerMaxPasses * 8);
    const int smem = kLayerWarps * d * kLayerStage<FULL> + p.room * row + rest;
    if (p.room < p.per) return err(WS_ERR_CAPACITY, "rows of %d activations do not fit", p.k);
    return d == 6 ? launch_layer<FIRST, PAIR, FULL, NT, 6>(err, p, smem, stream) : d == 4 ? launch_layer<FIRST, PAIR, FULL, NT, 4>(err, p, smem, stream)
                                                                                          : launch_layer<FIRST, PAIR, FULL, NT, 3>(err, p, smem, stream);
}
static_assert(kLayerWarps * 3 * kLayerStage<false> + 2 * layer_column_pitch(kLayerMaxWidth) + 2 * kLayerWarps * 2 * 4 * 32 * 4 <= kLayerSmem, "the widest rows");

int64_t layer_bytes(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" {

ws_status_t ws_head_norm_rope(const ws_head_norm_rope_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    if (a->m < 0 || a->q_heads < 0 || (a->k && a->k_heads < 0) || a->d < 1 || a->d > (1 << 24)) return err(WS_ERR_INVALID, "m=%d heads=%d,%d d=%d out of range", a->m, a->q_heads, a->k_heads, a->d);
    if (a->pairs < 0 || a->start < 0 || (int64_t)a->start + 2 * (int64_t)a->pairs > a->d) return err(WS_ERR_INVALID, "%d pairs from %d on are not within %d values", a->pairs, a->start, a->d);
    if (a->pairs > WS_MAX_PAIRS) return err(WS_ERR_CAPACITY, "%d pairs: at most %d", a->pairs, WS_MAX_PAIRS);
    if (!is_type(a->dtype) || !is_type(a->weight_dtype) || (a->position_bytes != 4 && a->position_bytes != 8)) return err(WS_ERR_INVALID, "unknown type of a tensor");
    if (!(a->eps >= 0.0f)) return err(WS_ERR_INVALID, "eps must not be negative");
    const int kh = a->k ? a->k_heads : 0;
    if ((int64_t)a->q_heads + kh > (1 << 24)) return err(WS_ERR_INVALID, "%d and %d heads: too many", a->q_heads, kh);
    if (a->m == 0 || a->q_heads + kh == 0) return WS_OK;
    if ((a->q_heads && (!a->q || !a->q_out)) || (kh && !a->k_out) || (a->pairs && (!a->positions || !a->inv_freq))) return err(WS_ERR_INVALID, "a tensor is missing");
    if (!natural(a->q, a->dtype) || !natural(a->k, a->dtype) || !natural(a->q_out, a->dtype) || !natural(a->k_out, a->dtype) || !natural(a->q_weight, a->weight_dtype) ||
        !natural(a->k_weight, a->weight_dtype) || (a->pairs && (!aligned_to(a->positions, a->position_bytes) || !aligned_to(a->inv_freq, 4))))
        return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    HeadsParams p{};
    p.x[0] = a->q; p.x[1] = a->k; p.y[0] = a->q_out; p.y[1] = a->k_out; p.w[0] = a->q_weight; p.w[1] = a->k_weight;
    p.ldt[0] = a->ldqt; p.ldt[1] = a->ldkt; p.ldh[0] = a->ldqh; p.ldh[1] = a->ldkh;
    p.ldyt[0] = a->ldqt_out; p.ldyt[1] = a->ldkt_out; p.ldyh[0] = a->ldqh_out; p.ldyh[1] = a->ldkh_out;
    p.heads[0] = a->q_heads; p.heads[1] = kh;
    p.positions = a->positions; p.inv_freq = a->inv_freq;
    p.m = a->m; p.d = a->d; p.pairs = a->pairs; p.start = a->start; p.interleaved = a->interleaved != 0; p.norm = a->norm != 0;
    p.dtype = a->dtype; p.w_dtype = a->weight_dtype; p.position_bytes = a->position_bytes;
    p.eps = a->eps; p.weight_offset = a->weight_offset; p.scale = a->scale;
    const int64_t eight = 8 * type_bytes(a->dtype);
    bool vec = a->d % 8 == 0 && a->start % 8 == 0 && (a->interleaved ? 2 * a->pairs : a->pairs) % 8 == 0 && a->d <= 2048;
    for (int i = 0; i < 2 && vec; ++i)
        if (p.heads[i])
            vec = aligned(p.x[i], p.ldt[i], a->dtype, eight) && aligned(p.x[i], p.ldh[i], a->dtype, eight) && aligned(p.y[i], p.ldyt[i], a->dtype, eight) &&
                  aligned(p.y[i], p.ldyh[i], a->dtype, eight) && aligned_to(p.w[i], 8 * type_bytes(a->weight_dtype));
    // units of two vectors (the part that is not rotated may have an odd one)
    const int halves = a->interleaved ? 0 : a->pairs / 8, all = halves + (a->d / 8 - 2 * halves + 1) / 2;
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes < all) p.lanes *= 2;
    const bool whole = all == p.lanes && a->d % 16 == 0;
    const int nu = (all + p.lanes - 1) / p.lanes, per = kHeadsThreads / (vec ? p.lanes : 32);
    // A token's heads go to several blocks where tokens are few; where they are many, a block takes four, so that a lane has
    // more heads for what it keeps of a token (64 + 8 heads of 128, one token a block and four: 300 tokens 5.3 and 6.8 us, 600 tokens
    // 9.0 and 8.7, 1184 tokens 13.5 and 10.6, 8192 tokens 90 and 61).
    const int rounds = (std::max(p.heads[0], p.heads[1]) + per - 1) / per;
    p.groups = p.teams = 1;
    while (p.groups < rounds && (int64_t)p.m * p.groups < 296) ++p.groups;
    if (vec && p.m >= 4 * 296 && 4 * p.pairs <= WS_MAX_PAIRS) p.teams = 4;
    if ((int64_t)p.m * p.groups > INT32_MAX) return err(WS_ERR_INVALID, "m=%d out of range", a->m);
    if (!vec) return launch(err, heads_any_kernel, dim3((unsigned)p.m * p.groups), kHeadsThreads, 0, 1, stream, p);
    return a->dtype == WS_ACT_F32 ? launch_heads<true>(err, nu, whole, p, stream) : launch_heads<false>(err, nu, whole, p, stream);
}

ws_status_t ws_moe_route(const ws_moe_route_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    if (a->m < 0 || a->experts < 1 || a->top_k < 1 || a->top_k > a->experts) return err(WS_ERR_INVALID, "m=%d experts=%d top_k=%d out of range", a->m, a->experts, a->top_k);
    if (a->experts > WS_ROUTE_MAX_EXPERTS || a->top_k > WS_ROUTE_MAX_TOP_K) return err(WS_ERR_CAPACITY, "%d of %d experts: at most %d of %d", a->top_k, a->experts, WS_ROUTE_MAX_TOP_K, WS_ROUTE_MAX_EXPERTS);
    if (!is_type(a->dtype) || a->score < WS_SCORE_SOFTMAX || a->score > WS_SCORE_SQRTSOFTPLUS) return err(WS_ERR_INVALID, "unknown type of a tensor or of the score");
    if (a->m == 0) return WS_OK;
    if (!a->logits || !a->ids || !a->weights) return err(WS_ERR_INVALID, "a tensor is missing");
    if (a->ld < a->experts) return err(WS_ERR_INVALID, "the row stride %lld is shorter than the row of %d values", (long long)a->ld, a->experts);
    if (!natural(a->logits, a->dtype) || !aligned_to(a->bias, 4) || !aligned_to(a->ids, 4) || !aligned_to(a->weights, 4)) return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    RouteParams p{};
    p.logits = a->logits; p.bias = a->bias; p.ld = a->ld; p.ids = a->ids; p.weights = a->weights;
    p.m = a->m; p.experts = a->experts; p.top_k = a->top_k; p.score = a->score; p.dtype = a->dtype; p.renormalize = a->renormalize; p.scale = a->scale;
    const dim3 grid((unsigned)(((int64_t)a->m + kRouteThreads / 32 - 1) / (kRouteThreads / 32)));
    const int n = (a->experts + 31) / 32;
    return a->dtype == WS_ACT_F32 ? launch_route<true>(err, n, grid, stream, p) : launch_route<false>(err, n, grid, stream, p);
}

int64_t ws_moe_layer_workspace(int32_t m, int32_t top_k, int32_t hidden, int32_t inter) {   // hidden of the routes, their results
    if (m < 1 || top_k < 1 || hidden < 1 || inter < 1) return 0;
    return layer_bytes((int64_t)m * top_k * inter * 4) + layer_bytes((int64_t)m * top_k * hidden * 4);
}

ws_status_t ws_moe_layer(const ws_moe_layer_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    if (a->m < 0 || a->top_k < 1 || a->hidden < 32 || a->inter < 32 || a->hidden % 32 || a->inter % 32)
        return err(WS_ERR_INVALID, "m=%d top_k=%d hidden=%d inter=%d: widths are multiples of 32", a->m, a->top_k, a->hidden, a->inter);
    if (a->e_len < 1 || a->e_start < 0) return err(WS_ERR_INVALID, "bad local expert range");
    if (!is_type(a->x_dtype) || !is_type(a->out_dtype)) return err(WS_ERR_INVALID, "unknown type of a tensor");
    if (a->limit != a->limit) return err(WS_ERR_INVALID, "limit is no number");
    if (a->top_k > kLayerMaxTopK || (int64_t)a->m * a->top_k > kLayerMaxRoutes) return err(WS_ERR_CAPACITY, "m*top_k = %d*%d exceeds %d routes per call", a->m, a->top_k, kLayerMaxRoutes);
    if (a->e_len > kLayerMaxExperts || a->hidden > kLayerMaxWidth || a->inter > kLayerMaxWidth)
        return err(WS_ERR_CAPACITY, "%d experts of %d x %d: at most %d of %d", a->e_len, a->hidden, a->inter, kLayerMaxExperts, kLayerMaxWidth);
    if (a->m == 0) return WS_OK;
    if (!a->x || !a->route_ids || !a->route_w || !a->w1 || !a->s1 || !a->w3 || !a->s3 || !a->w2 || !a->s2 || !a->out) return err(WS_ERR_INVALID, "a tensor is missing");
    if (a->ldx < a->hidden || a->ldo < a->hidden) return err(WS_ERR_INVALID, "a row stride is shorter than its row");
    const void *const w[6] = {a->w1, a->s1, a->w3, a->s3, a->w2, a->s2};
    const int64_t stride[6] = {a->w1_stride, a->s1_stride, a->w3_stride, a->s3_stride, a->w2_stride, a->s2_stride};
    for (int i = 0; i < 6; ++i)
        if (!aligned_to(w[i], 16) || stride[i] % 16 || stride[i] < (int64_t)a->hidden * a->inter / (i % 2 ? 32 : 2))
            return err(WS_ERR_INVALID, "weights and scales are 16-byte aligned, their experts multiples of 16 bytes apart and not within one another");
    if (!natural(a->x, a->x_dtype) || !natural(a->out, a->out_dtype) || !aligned_to(a->route_ids, 4) || !aligned_to(a->route_w, 4)) return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    const int64_t need = ws_moe_layer_workspace(a->m, a->top_k, a->hidden, a->inter);
    if (!a->workspace || a->workspace_bytes < need || !aligned_to(a->workspace, 16)) return err(WS_ERR_INVALID, "a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
    LayerParams p{};
    char *work = static_cast<char *>(a->workspace);
    p.h = reinterpret_cast<float *>(work); work += layer_bytes((int64_t)a->m * a->top_k * a->inter * 4);
    p.part = reinterpret_cast<float *>(work);
    p.x = a->x; p.ldx = a->ldx; p.x_dtype = a->x_dtype; p.vec = aligned(a->x, a->ldx, a->x_dtype, 16);
    p.ids = a->route_ids; p.weights = a->route_w; p.m = a->m; p.top_k = a->top_k; p.e_start = a->e_start; p.e_len = a->e_len;
    p.out = a->out; p.ldo = a->ldo; p.out_dtype = a->out_dtype; p.act_quant = a->act_quant != 0;
    p.has_limit = a->limit > 0.0f; p.limit = a->limit;
    LayerParams q = p;
    p.wa = a->w1; p.sa = a->s1; p.wb = a->w3; p.sb = a->s3;
    p.wa_e = a->w1_stride; p.sa_e = a->s1_stride; p.wb_e = a->w3_stride; p.sb_e = a->s3_stride;
    p.k = a->hidden; p.units = a->inter / 8; p.n = a->inter;
    q.wa = q.wb = a->w2; q.sa = q.sb = a->s2; q.wa_e = q.wb_e = a->w2_stride; q.sa_e = q.sb_e = a->s2_stride;
    q.k = a->inter; q.units = a->hidden / 32; q.n = a->hidden;
    const bool pair = a->x_dtype == WS_ACT_F32 && !a->act_quant, full = p.k % kLayerChunk == 0;
    ws_status_t st = pair ? full ? launch_layer<true, true, true, 1>(err, p, stream) : launch_layer<true, true, false, 1>(err, p, stream)
                          : full ? launch_layer<true, false, true, 1>(err, p, stream) : launch_layer<true, false, false, 1>(err, p, stream);
    if (st != WS_OK) return st;
    // (Eight columns or sixteen, us: 12 tokens of 7168 x 2048 by 4 of 24 experts
    // 120 and 124, 16 tokens of 1024 x 512 by 8 of 64 28.7 and 33.8, 64 tokens of 2048 x 768 by 8 of 128 91.5 and 89.)
    if (q.k % kLayerChunk == 0) st = a->m <= 4 ? launch_layer<false, true, true, 1>(err, q, stream) : launch_layer<false, true, true, 2>(err, q, stream);
    else st = a->m <= 4 ? launch_layer<false, true, false, 1>(err, q, stream) : launch_layer<false, true, false, 2>(err, q, stream);
    if (st != WS_OK) return st;
    q.vec = aligned(a->out, a->ldo, a->out_dtype, 4 * type_bytes(a->out_dtype));
    return launch(err, layer_sum_kernel, dim3((unsigned)(((int64_t)a->m * (a->hidden / 4) + kLayerSumThreads - 1) / kLayerSumThreads)), kLayerSumThreads, 0, 1, stream, q);
}

ws_status_t ws_adjust_logits(const ws_adjust_logits_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    // (the kernel counts a row's values in 32 bits, up to a slice past its end)
    if (a->m < 0 || a->vocab < 1 || a->vocab > INT32_MAX - (1 << 16)) return err(WS_ERR_INVALID, "m=%d vocab=%d out of range", a->m, a->vocab);
    if (!is_type(a->dtype)) return err(WS_ERR_INVALID, "unknown type of a tensor");
    auto width = [](int32_t b) { return b == 4 || b == 8; };
    if ((a->tokens && !width(a->offset_bytes)) || (a->bias_ids && !width(a->bias_offset_bytes))) return err(WS_ERR_INVALID, "unknown type of a tensor");
    if (a->n_tokens < 0 || a->n_bias < 0 || a->n_bias > INT32_MAX || a->mask_count < 0) return err(WS_ERR_INVALID, "sizes of tokens, biases or masks out of range");
    if (a->m == 0) return WS_OK;
    if (!a->logits || !a->out || (a->tokens && !a->offsets) || (a->bias_ids && (!a->bias || !a->bias_offsets))) return err(WS_ERR_INVALID, "a tensor is missing");
    if (a->ld < a->vocab || a->ldo < a->vocab || (a->mask && a->ld_mask < ((int64_t)a->vocab + 31) / 32)) return err(WS_ERR_INVALID, "a row stride is shorter than its row");
    if (!natural(a->logits, a->dtype) || !natural(a->out, a->dtype) || !aligned_to(a->tokens, 4) || !aligned_to(a->prompt_lens, 4) || !aligned_to(a->repetition, 4) ||
        !aligned_to(a->frequency, 4) || !aligned_to(a->presence, 4) || !aligned_to(a->bias_ids, 4) || !aligned_to(a->bias, 4) || !aligned_to(a->mask, 4) ||
        !aligned_to(a->mask_rows, 4) || (a->tokens && !aligned_to(a->offsets, a->offset_bytes)) || (a->bias_ids && !aligned_to(a->bias_offsets, a->bias_offset_bytes)))
        return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    AdjustParams p{};
    p.logits = a->logits; p.out = a->out; p.ld = a->ld; p.ldo = a->ldo; p.m = a->m; p.vocab = a->vocab;
    if (a->tokens) {
        p.tokens = a->tokens; p.offsets = a->offsets; p.offset_bytes = a->offset_bytes; p.n_tokens = a->n_tokens; p.prompt_lens = a->prompt_lens;
        p.repetition = a->repetition; p.frequency = a->frequency; p.presence = a->presence;
    }
    if (a->bias_ids) { p.bias_ids = a->bias_ids; p.bias = a->bias; p.bias_offsets = a->bias_offsets; p.bias_offset_bytes = a->bias_offset_bytes; p.n_bias = a->n_bias; }
    if (a->mask) { p.mask = a->mask; p.mask_rows = a->mask_rows; p.mask_count = a->mask_count; p.ld_mask = a->ld_mask; }
    const int64_t es = type_bytes(a->dtype);
    // a row's values and results lie alike within 16 bytes
    const bool vec = (reinterpret_cast<uintptr_t>(a->logits) - reinterpret_cast<uintptr_t>(a->out)) % 16 == 0 && (a->ld - a->ldo) * es % 16 == 0;
    p.in_place = a->logits == a->out && a->ld == a->ldo;
    if (p.in_place && !p.mask && !p.tokens && !p.bias_ids) return WS_OK;
    if (a->dtype == WS_ACT_F32) return vec ? launch_adjust<true, true>(err, p, stream) : launch_adjust<true, false>(err, p, stream);
    return vec ? launch_adjust<false, true>(err, p, stream) : launch_adjust<false, false>(err, p, stream);
}

}  // extern "C"
