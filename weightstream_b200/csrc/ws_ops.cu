// C entry points of the operators between the tensor-parallel steps (include/ws_tp.h): checks of arguments, choice of
// kernel, launch.
#include <algorithm>

#include "ws_lora_kernel.cuh"
#include "ws_norm_kernel.cuh"
#include "ws_ops_host.cuh"
#include "ws_scores_kernel.cuh"

using namespace ws;

namespace {

// ---- norms
template <int NV, bool VEC, bool YF32, int RK>
ws_status_t launch_norm(const Err &err, const NormParams &p, void *stream) {
    const unsigned threads = (unsigned)((p.n + NV * 8 * 32 - 1) / (NV * 8 * 32)) * 32;
    const int gk = !p.gate || !p.gate_inc ? 0 : p.g_dtype == WS_ACT_F32 ? 2 : 1;
    auto *k = gk == 0 ? block_norm_rows_kernel<NV, VEC, YF32, RK, 0> : gk == 1 ? block_norm_rows_kernel<NV, VEC, YF32, RK, 1>
                                                                              : block_norm_rows_kernel<NV, VEC, YF32, RK, 2>;
    return launch(err, k, dim3((unsigned)p.m), threads, 0, 1, stream, p);
}
template <int NV, bool VEC, bool YF32>
ws_status_t launch_norm(const Err &err, const NormParams &p, void *stream) {
    if (!p.residual) return launch_norm<NV, VEC, YF32, 0>(err, p, stream);
    return p.r_dtype == WS_ACT_F32 ? launch_norm<NV, VEC, YF32, 2>(err, p, stream) : launch_norm<NV, VEC, YF32, 1>(err, p, stream);
}
template <int NV, bool VEC>
ws_status_t launch_norm(const Err &err, const NormParams &p, void *stream) {
    return p.y_dtype == WS_ACT_F32 ? launch_norm<NV, VEC, true>(err, p, stream) : launch_norm<NV, VEC, false>(err, p, stream);
}
ws_status_t norm(const Err &err, const NormParams &p, void *stream) {
    auto wide = [](const void *q, int64_t ld, int32_t type) { return !q || aligned(q, ld, type, 8 * type_bytes(type)); };
    const bool vec = p.n % 8 == 0 && wide(p.y, p.ldy, p.y_dtype) && wide(p.residual, p.ldr, p.r_dtype) && (!p.gate_inc || wide(p.gate, p.ldg, p.g_dtype)) &&
                     wide(p.post_weight, 0, p.w_dtype) && wide(p.next_weight, 0, p.w_dtype) && wide(p.hidden, p.ldh, p.h_dtype) && wide(p.normed, p.ldn, p.n_dtype);
    // Eight values a thread where rows are few or short (one row 2.7 us against 3.1 with sixteen, 1503 rows of 2307 11.0 us
    // against 11.4); sixteen keep more blocks an SM loading while others sum (8192 rows of 7168 124 us against 186, with 32
    // 155); wider rows need more registers a thread, up to 32 values.
    const int nv = p.n > 8192 ? 4 : p.m <= 296 || p.n <= 2560 ? 1 : 2;
    if (p.n > 16384) return launch(err, block_norm_any_kernel, dim3((unsigned)p.m), 512, 0, 1, stream, p);
    if (vec) return nv == 1 ? launch_norm<1, true>(err, p, stream) : nv == 2 ? launch_norm<2, true>(err, p, stream) : launch_norm<4, true>(err, p, stream);
    return nv == 1 ? launch_norm<1, false>(err, p, stream) : nv == 2 ? launch_norm<2, false>(err, p, stream) : launch_norm<4, false>(err, p, stream);
}

// ---- scores
template <int T, bool F32, bool TOP>
ws_status_t launch_scores(const Err &err, const ScoreParams &p, void *stream) {
    constexpr auto k = token_scores_kernel<T, F32, TOP>;
    const ws_status_t st = allow_smem<k>(err, kScoreSmem<T, F32>);
    return st != WS_OK ? st : launch(err, k, dim3((unsigned)p.m * p.cluster), T, kScoreSmem<T, F32>, (unsigned)p.cluster, stream, p);
}
template <int T>
ws_status_t launch_scores(const Err &err, bool f32, const ScoreParams &p, void *stream) {
    if (f32) return p.top ? launch_scores<T, true, true>(err, p, stream) : launch_scores<T, true, false>(err, p, stream);
    return p.top ? launch_scores<T, false, true>(err, p, stream) : launch_scores<T, false, false>(err, p, stream);
}

// ---- adapters
int64_t lora_max_tiles(int m, int adapters, int tile) { return ((int64_t)m + tile - 1) / tile + std::min((int64_t)adapters + 1, (int64_t)m); }
int64_t lora_perm_bytes(int m) { return 16 + ((int64_t)m * 4 + 15) / 16 * 16; }

template <int RT, int NT, bool XF32, bool VEC>
ws_status_t launch_lora(const Err &err, unsigned tiles, void *stream, const LoraParams &p) {
    using S = LoraShape<RT, NT>;
    constexpr auto k = lora_kernel<RT, NT, XF32, VEC>;
    if (S::kSmem > 47 * 1024) {  // (48 KB with the static part)
        const ws_status_t st = allow_smem<k>(err, S::kSmem);
        if (st != WS_OK) return st;
    }
    return launch(err, k, dim3(tiles * (unsigned)p.cluster), kLoraThreads, S::kSmem, (unsigned)p.cluster, stream, p);
}
template <int RT, int NT>
ws_status_t launch_lora(const Err &err, bool xf32, bool vec, unsigned tiles, void *stream, const LoraParams &p) {
    if (!vec) return xf32 ? launch_lora<RT, NT, true, false>(err, tiles, stream, p) : launch_lora<RT, NT, false, false>(err, tiles, stream, p);
    return xf32 ? launch_lora<RT, NT, true, true>(err, tiles, stream, p) : launch_lora<RT, NT, false, true>(err, tiles, stream, p);
}
template <int RT>
ws_status_t launch_lora(const Err &err, int nt, bool xf32, bool vec, unsigned tiles, void *stream, const LoraParams &p) {
    return nt == 1 ? launch_lora<RT, 1>(err, xf32, vec, tiles, stream, p) : launch_lora<RT, 2>(err, xf32, vec, tiles, stream, p);
}

template <int RT, bool XF32, bool VEC>
ws_status_t launch_shrink(const Err &err, unsigned tiles, void *stream, LoraParams &p) {
    constexpr auto k = lora_shrink_kernel<RT, XF32, VEC>;
    constexpr int smem = ShrinkShape<RT, XF32>::kSmem, at_once = 148 * kShrinkBlocks<RT, XF32, VEC>;
    // The device cuts K by the tiles that there are (lora_shrink_cut).  A cluster has the blocks of the largest cut, which is
    // that of all tiles that there can be, or of twice the fewest where a table has adapters for more.  A batch that may
    // have too many tiles for a cut gets a launch without clusters beside, and one of the two finds its work: blocks of
    // clusters of eight that each take a tile are placed worse (1000 tokens of 500 adapters, rank 128, 314 us; alone 242).
    const int fewest = (p.m + kSortTokens - 1) / kSortTokens, usual = std::min((int)tiles, 2 * fewest);
    p.most = 0;
    while (p.most < 3 && usual << p.most < 148 && p.k >> (p.most + 1) >= 2 * kSortK) ++p.most;
    ws_status_t st = allow_smem<k>(err, smem);
    if (st == WS_OK && p.most > 0) {
        p.cluster = 1 << p.most;
        const unsigned blocks = std::min(tiles << p.most, (unsigned)(at_once + fewest)), clusters = (blocks + p.cluster - 1) / p.cluster;
        st = launch(err, k, dim3(clusters * p.cluster), kLoraThreads, smem, (unsigned)p.cluster, stream, p);
    }
    if (st == WS_OK && (p.most == 0 || (int)tiles > at_once / 2)) {
        p.cluster = 1;
        st = launch(err, k, dim3(tiles), kLoraThreads, smem, 1, stream, p);
    }
    return st;
}
template <int RT>
ws_status_t launch_shrink(const Err &err, bool xf32, bool vec, unsigned tiles, void *stream, LoraParams &p) {
    if (vec) return xf32 ? launch_shrink<RT, true, true>(err, tiles, stream, p) : launch_shrink<RT, false, true>(err, tiles, stream, p);
    return xf32 ? launch_shrink<RT, true, false>(err, tiles, stream, p) : launch_shrink<RT, false, false>(err, tiles, stream, p);
}
template <int RT, bool YF32, bool VEC>
ws_status_t launch_expand(const Err &err, unsigned tiles, void *stream, const LoraParams &p) {
    constexpr auto k = lora_expand_kernel<RT, YF32, VEC>;
    constexpr int smem = ExpandShape<RT>::kSmem;
    const ws_status_t st = allow_smem<k>(err, smem);
    return st != WS_OK ? st : launch(err, k, dim3(tiles * (unsigned)p.cluster), kLoraThreads, smem, 1, stream, p);
}
template <int RT>
ws_status_t launch_expand(const Err &err, bool vec, unsigned tiles, void *stream, const LoraParams &p) {
    const bool yf32 = p.y_dtype == WS_ACT_F32;
    if (vec) return yf32 ? launch_expand<RT, true, true>(err, tiles, stream, p) : launch_expand<RT, false, true>(err, tiles, stream, p);
    return yf32 ? launch_expand<RT, true, false>(err, tiles, stream, p) : launch_expand<RT, false, false>(err, tiles, stream, p);
}

enum class Lora { kAdd, kShrink, kExpand };

ws_status_t lora(Lora what, const ws_lora_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    const bool shrinks = what != Lora::kExpand, expands = what != Lora::kShrink;
    // (the kernels count a row's values in 32 bits, up to a step past its end, and blocks in 31)
    if (a->m < 0 || a->m > (1 << 26) || a->adapters < 1 || (shrinks && (a->k < 1 || a->k > INT32_MAX - 4096)) ||
        (expands && (a->n < 1 || a->n > INT32_MAX - 4096)))
        return err(WS_ERR_INVALID, "m=%d k=%d n=%d adapters=%d out of range", a->m, a->k, a->n, a->adapters);
    if (a->rank < 1 || a->rank > WS_LORA_MAX_RANK) return err(WS_ERR_INVALID, "rank=%d is not in 1..%d", a->rank, WS_LORA_MAX_RANK);
    if ((shrinks && !is_type(a->x_dtype)) || (expands && !is_type(a->y_dtype))) return err(WS_ERR_INVALID, "unknown type of a tensor");
    if (a->m == 0) return WS_OK;
    if (!a->ids || (shrinks && (!a->x || !a->a)) || (expands && (!a->y || !a->out || !a->b)) || (what != Lora::kAdd && !a->shrunk))
        return err(WS_ERR_INVALID, "a tensor is missing");
    if ((shrinks && a->ldx < a->k) || (expands && (a->ldy < a->n || a->ldo < a->n))) return err(WS_ERR_INVALID, "a row stride is shorter than its row");
    if ((shrinks && (!natural(a->x, a->x_dtype) || !natural(a->a, WS_ACT_BF16))) ||
        (expands && (!natural(a->y, a->y_dtype) || !natural(a->out, a->y_dtype) || !natural(a->b, WS_ACT_BF16))) ||
        !natural(a->ids, WS_ACT_F32) || !natural(a->scale, WS_ACT_F32) || !natural(a->shrunk, WS_ACT_F32))
        return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    LoraParams p{};
    if (shrinks) { p.x = a->x; p.a = static_cast<const uint16_t *>(a->a); p.ldx = a->ldx; p.k = a->k; }
    if (expands) { p.y = a->y; p.out = a->out; p.b = static_cast<const uint16_t *>(a->b); p.ldy = a->ldy; p.ldo = a->ldo; p.n = a->n; p.scale = a->scale; p.y_dtype = a->y_dtype; }
    if (what == Lora::kShrink) p.s_out = a->shrunk;
    if (what == Lora::kExpand) p.s_in = a->shrunk;
    p.ids = a->ids; p.m = a->m; p.r = a->rank; p.adapters = a->adapters;
    p.skip_none = expands && a->y == a->out && a->ldy == a->ldo;
    const bool xf32 = shrinks && a->x_dtype == WS_ACT_F32;
    // whole vectors of ranks; of K; of N
    const bool vec_r = a->rank % 8 == 0 && (!expands || aligned(a->b, a->rank, WS_ACT_BF16, 16));
    bool vec_k = true, vec_n = true;
    if (shrinks) vec_k = a->k % 8 == 0 && aligned(a->x, a->ldx, a->x_dtype, 16) && aligned(a->a, a->k, WS_ACT_BF16, 16);
    if (expands) {
        const int64_t four = 4 * type_bytes(a->y_dtype);
        vec_n = a->n % 4 == 0 && aligned(a->y, a->ldy, a->y_dtype, four) && aligned(a->out, a->ldo, a->y_dtype, four);
    }
    const bool vec = vec_r && vec_k && vec_n;
    const int rt = a->rank <= 16 ? 1 : a->rank <= 32 ? 2 : a->rank <= 64 ? 4 : 8;
    const int nt = a->m <= 128 ? 1 : 2;
    unsigned tiles = (unsigned)std::min((int64_t)a->m, lora_max_tiles(a->m, a->adapters, nt * 8));
    p.cluster = tiles <= 148 ? 8 : 4;  // (333 rows of up to 54 tiles 14.8 us with 8 blocks a tile, 17.4 with 4)
    if (a->m > kLoraDirect) {
        const int64_t need = ws_lora_workspace(a->m, a->adapters, a->rank);
        if (a->adapters > kLoraMaxAdapters) return err(WS_ERR_CAPACITY, "%d adapters: at most %d with more than %d tokens", a->adapters, kLoraMaxAdapters, kLoraDirect);
        if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) & 15)
            return err(WS_ERR_INVALID, "%d tokens need a 16-byte aligned workspace of %lld bytes", a->m, (long long)need);
        p.tile = vec_r ? kSortTokens : nt * 8;
        p.tiles_count = static_cast<int32_t *>(a->workspace);
        p.perm = p.tiles_count + 4;
        p.tiles = reinterpret_cast<LoraTile *>(static_cast<char *>(a->workspace) + lora_perm_bytes(a->m));
        tiles = (unsigned)lora_max_tiles(a->m, a->adapters, p.tile);
        const size_t smem = (size_t)(a->adapters + 1) * 12;
        if (smem > 47 * 1024) {
            const ws_status_t st = allow_smem<lora_plan_kernel>(err, (kLoraMaxAdapters + 1) * 12);
            if (st != WS_OK) return st;
        }
        ws_status_t st = launch(err, lora_plan_kernel, dim3(1), 1024, smem, 1, stream, p);
        if (st != WS_OK) return st;
        if (vec_r) {
            if (shrinks) {
                LoraParams q = p;
                if (expands) q.s_out = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + need) - (int64_t)a->m * a->rank;
                p.s_in = expands ? q.s_out : nullptr;
                q.skip_none = 0;
                st = rt == 1 ? launch_shrink<1>(err, xf32, vec_k, tiles, stream, q) : rt == 2 ? launch_shrink<2>(err, xf32, vec_k, tiles, stream, q)
                     : rt == 4 ? launch_shrink<4>(err, xf32, vec_k, tiles, stream, q) : launch_shrink<8>(err, xf32, vec_k, tiles, stream, q);
                if (st != WS_OK || !expands) return st;
            }
            // N is cut so that the slices' blocks, one an SM from rank 33 and two below, end together with the tiles that there
            // may well be (rank 64, 4000 rows: 113 us with 2 slices, 122 with 4; rank 16, 2000 rows: 70 us with 4, 48 with 8)
            const int64_t likely = (a->m + kSortTokens - 1) / kSortTokens + std::min(a->adapters, a->m / kSortTokens) / 2, at_once = rt >= 4 ? 148 : 296;
            const int rounds = (a->n + kExpandN - 1) / kExpandN;
            int64_t least = INT64_MAX;
            for (int c = 1; c <= rounds && c <= 32; ++c) {  // (a block's beginning costs about one round)
                const int64_t cost = (likely * c + at_once - 1) / at_once * ((rounds + c - 1) / c + 1);
                if (cost < least) {
                    least = cost;
                    p.cluster = c;
                }
            }
            return rt == 1 ? launch_expand<1>(err, vec_n, tiles, stream, p) : rt == 2 ? launch_expand<2>(err, vec_n, tiles, stream, p)
                   : rt == 4 ? launch_expand<4>(err, vec_n, tiles, stream, p) : launch_expand<8>(err, vec_n, tiles, stream, p);
        }
    }
    switch (rt) {
        case 1: return launch_lora<1>(err, nt, xf32, vec, tiles, stream, p);
        case 2: return launch_lora<2>(err, nt, xf32, vec, tiles, stream, p);
        case 4: return launch_lora<4>(err, nt, xf32, vec, tiles, stream, p);
        default: return launch_lora<8>(err, nt, xf32, vec, tiles, stream, p);
    }
}

}  // namespace

extern "C" {

int64_t ws_lora_workspace(int32_t m, int32_t adapters, int32_t rank) {  // plan, then shrunk rows
    if (m <= kLoraDirect || adapters < 1 || rank < 1) return 0;
    return lora_perm_bytes(m) + lora_max_tiles(m, adapters, 16) * (int64_t)sizeof(LoraTile) + ((int64_t)m * rank * 4 + 15) / 16 * 16;
}
ws_status_t ws_lora_add(const ws_lora_args_t *a, void *stream, char *err, size_t err_len) { return lora(Lora::kAdd, a, stream, err, err_len); }
ws_status_t ws_lora_shrink(const ws_lora_args_t *a, void *stream, char *err, size_t err_len) { return lora(Lora::kShrink, a, stream, err, err_len); }
ws_status_t ws_lora_expand(const ws_lora_args_t *a, void *stream, char *err, size_t err_len) { return lora(Lora::kExpand, a, stream, err, err_len); }


ws_status_t ws_block_norm(const ws_block_norm_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    // (the kernels count a row's values in 32 bits, up to a step past its end)
    if (a->m < 0 || a->n < 1 || a->n > INT32_MAX - 4096) return err(WS_ERR_INVALID, "m=%d n=%d out of range", a->m, a->n);
    if (!is_type(a->y_dtype) || !is_type(a->residual_dtype) || !is_type(a->gate_dtype) || !is_type(a->weight_dtype) ||
        !is_type(a->hidden_dtype) || !is_type(a->normed_dtype))
        return err(WS_ERR_INVALID, "unknown type of a tensor");
    if (a->gate_inc < 0 || a->gate_inc > 1 || (a->gate_act != WS_GATE_LINEAR && a->gate_act != WS_GATE_SIGMOID))
        return err(WS_ERR_INVALID, "gate_inc=%d gate_act=%d: unknown form of the gate", a->gate_inc, a->gate_act);
    if (!(a->eps >= 0.0f)) return err(WS_ERR_INVALID, "eps must not be negative");
    if (a->m == 0) return WS_OK;
    if (!a->y || (!a->hidden && !a->normed)) return err(WS_ERR_INVALID, "y and one of hidden and normed are needed");
    if (a->normed && !a->next_weight) return err(WS_ERR_INVALID, "normed needs next_weight");
    if (a->ldy < a->n || (a->residual && a->ldr < a->n) || (a->hidden && a->ldh < a->n) || (a->normed && a->ldn < a->n) || (a->gate && a->ldg < 0))
        return err(WS_ERR_INVALID, "a row stride is shorter than the row of %d values", a->n);
    if (!natural(a->y, a->y_dtype) || !natural(a->residual, a->residual_dtype) || !natural(a->gate, a->gate_dtype) ||
        !natural(a->post_weight, a->weight_dtype) || !natural(a->next_weight, a->weight_dtype) || !natural(a->hidden, a->hidden_dtype) ||
        !natural(a->normed, a->normed_dtype))
        return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    NormParams p{};
    p.y = a->y; p.residual = a->residual; p.gate = a->gate; p.post_weight = a->post_weight; p.next_weight = a->next_weight;
    p.hidden = a->hidden; p.normed = a->normed;
    p.ldy = a->ldy; p.ldr = a->ldr; p.ldg = a->ldg; p.ldh = a->ldh; p.ldn = a->ldn;
    p.m = a->m; p.n = a->n; p.gate_inc = a->gate_inc; p.gate_act = a->gate_act;
    p.y_dtype = a->y_dtype; p.r_dtype = a->residual_dtype; p.g_dtype = a->gate_dtype; p.w_dtype = a->weight_dtype;
    p.h_dtype = a->hidden_dtype; p.n_dtype = a->normed_dtype;
    p.weight_offset = a->weight_offset; p.eps = a->eps; p.residual_scale = a->residual_scale; p.block_scale = a->block_scale;
    return norm(err, p, stream);
}

ws_status_t ws_token_logprobs(const ws_token_logprobs_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    // (the kernel counts a row's values in 32 bits, up to a vector and a batch of vectors past its end)
    if (a->m < 0 || a->m > INT32_MAX / kScoreMaxCluster || a->vocab < 1 || a->vocab > INT32_MAX - (1 << 16))
        return err(WS_ERR_INVALID, "m=%d vocab=%d out of range", a->m, a->vocab);
    if (a->top < 0 || a->top > WS_MAX_TOP) return err(WS_ERR_INVALID, "top=%d is not in 0..%d", a->top, WS_MAX_TOP);
    if (!is_type(a->dtype) || (a->token_bytes != 4 && a->token_bytes != 8)) return err(WS_ERR_INVALID, "unknown type of a tensor");
    if (a->m == 0) return WS_OK;
    if (!a->logits || !a->tokens || !a->logprob || !a->entropy || !a->rank || (a->top && (!a->top_id || !a->top_logprob)))
        return err(WS_ERR_INVALID, "a tensor is missing");
    if (a->ld < a->vocab) return err(WS_ERR_INVALID, "the row stride %lld is shorter than the row of %d values", (long long)a->ld, a->vocab);
    if (!natural(a->logits, a->dtype) || reinterpret_cast<uintptr_t>(a->tokens) % a->token_bytes || !natural(a->logprob, WS_ACT_F32) ||
        !natural(a->entropy, WS_ACT_F32) || !natural(a->rank, WS_ACT_F32) ||
        (a->top && (!natural(a->top_id, WS_ACT_F32) || !natural(a->top_logprob, WS_ACT_F32))))
        return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    ScoreParams p{};
    p.logits = a->logits; p.tokens = a->tokens; p.ld = a->ld; p.m = a->m; p.vocab = a->vocab; p.top = a->top; p.token_bytes = a->token_bytes;
    p.logprob = a->logprob; p.entropy = a->entropy; p.top_logprob = a->top_logprob; p.rank = a->rank; p.top_id = a->top_id;
    // Few rows: a row is cut over a cluster, as long as two blocks an SM take them all (64 rows: 17 us with four blocks a
    // row, 23 with two, 29 with eight) and a thread of each has a vector.  Blocks of 512 threads then have the shorter way
    // (one row 9 us against 12, 64 rows 17 against 21); smaller blocks, three or four an SM, lose less while one of them
    // ranks its alternatives (2000 rows with 20 of them 190 us against 217, without them 160 against 161).
    const int vector = a->dtype == WS_ACT_F32 ? 4 : 8;
    int c = 1;
    while (c < 8 && (int64_t)a->m * c * 2 <= 320 && a->vocab / (2 * c) >= vector * 256) c *= 2;
    p.cluster = c;
    const int t = (int64_t)a->m * c <= 296 ? 512 : 256;
    return t == 512 ? launch_scores<512>(err, a->dtype == WS_ACT_F32, p, stream) : launch_scores<256>(err, a->dtype == WS_ACT_F32, p, stream);
}

}  // extern "C"
