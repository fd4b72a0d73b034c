// C entry points of the operators between the tensor-parallel steps (include/ws_tp.h): checks of arguments, choice of
// kernel, launch.
#include <algorithm>
#include <cstdarg>
#include <cstdio>

#include "ws_norm_kernel.cuh"
#include "ws_scores_kernel.cuh"

using namespace ws;

namespace {

struct Err {  // the caller's message buffer
    char *p;
    size_t len;
    ws_status_t operator()(ws_status_t st, const char *fmt, ...) const {
        if (p && len) {
            va_list ap;
            va_start(ap, fmt);
            vsnprintf(p, len, fmt, ap);
            va_end(ap);
        }
        return st;
    }
};

bool is_type(int32_t t) { return t == WS_ACT_BF16 || t == WS_ACT_F32; }
int64_t type_bytes(int32_t t) { return t == WS_ACT_BF16 ? 2 : 4; }
bool aligned(const void *p, int64_t ld, int32_t type, int64_t bytes) {  // first values of all rows
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * type_bytes(type) % bytes == 0;
}
bool natural(const void *p, int32_t type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0; }

// The kernels begin with griddepcontrol.wait, so their launch may overlap the end of the kernel before them.
template <typename P>
ws_status_t launch(const Err &err, void (*kernel)(P), dim3 grid, unsigned threads, size_t smem, unsigned cluster, void *stream, const P &params) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params);
    return e == cudaSuccess ? WS_OK : err(WS_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
}

}  // namespace

extern "C" {

ws_status_t ws_block_norm(const ws_block_norm_args_t *a, void *stream, char *err_text, size_t err_len) {
    const Err err{err_text, err_len};
    if (err_text && err_len) err_text[0] = 0;
    if (!a) return err(WS_ERR_INVALID, "null args");
    if (a->m < 0 || a->n < 1) return err(WS_ERR_INVALID, "m=%d n=%d: m must not be negative, n at least 1", a->m, a->n);
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
    const unsigned threads = (unsigned)std::min(512, (p.n + 31) / 32 * 32);
    return launch(err, block_norm_any_kernel, dim3((unsigned)p.m), threads, 0, 1, stream, p);
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
    if (!natural(a->logits, a->dtype) || reinterpret_cast<uintptr_t>(a->tokens) % a->token_bytes)
        return err(WS_ERR_INVALID, "a tensor is not aligned to its type");
    ScoreParams p{};
    p.logits = a->logits; p.tokens = a->tokens; p.ld = a->ld; p.m = a->m; p.vocab = a->vocab; p.top = a->top; p.token_bytes = a->token_bytes;
    p.logprob = a->logprob; p.entropy = a->entropy; p.top_logprob = a->top_logprob; p.rank = a->rank; p.top_id = a->top_id;
    const int per = (a->dtype == WS_ACT_F32 ? 4 : 8) * kScoreThreads;  // values of one round of a block
    int c = 1;
    while (c < kScoreMaxCluster && (int64_t)a->m * c * 2 <= 2 * 148 && a->vocab / (2 * c) >= per) c *= 2;
    p.cluster = c;
    const dim3 grid((unsigned)a->m * c);
    auto *k = a->dtype == WS_ACT_F32 ? (a->top ? token_scores_kernel<true, true> : token_scores_kernel<true, false>)
                                     : (a->top ? token_scores_kernel<false, true> : token_scores_kernel<false, false>);
    return launch(err, k, grid, kScoreThreads, 0, (unsigned)c, stream, p);
}

}  // extern "C"
