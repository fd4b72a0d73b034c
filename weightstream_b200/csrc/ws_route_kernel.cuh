// Experts of every token from the gate's logits: the top_k by  key = score + bias  (score alone without one), larger
// first and equal ones by index, and their weights  scale * score  or  scale * score / sum of the chosen scores.
//
//   score = softmax(l), sigmoid(l) or sqrt(ln(1 + e^l))
//
// A warp takes a token, its logits in registers.  Without a bias the order is that of the logits themselves.  With one,
// keys are compared in 32 bits first; where two neighbours of the order lie as close as their errors, the candidates'
// keys are taken again in 64 bits, so that the choice is the definition's and not that of a rounding.  Errors go by the
// largest score of the token, chosen or not: a bias may cancel a score of any size and leave its rounding.
// Experts whose logit is -inf or NaN are never chosen; places that stay empty hold id -1 and weight 0.
//
// Bound: instructions (4096 tokens of 384 experts with a bias, top 8: 19 to 21 us, 1600 of them
// a token; HBM would need 1), the launch for few (64 tokens 5.1 us a call).
#pragma once

#include "ws_values.cuh"

namespace ws {

constexpr int kRouteThreads = 128;
static_assert(WS_ROUTE_MAX_TOP_K == 32 && WS_ROUTE_MAX_EXPERTS <= 32 * 32, "a lane keeps one result, and 32 logits");
constexpr float kRouteNear = 4e-6f;     // keys that differ by less than this share of them, of the largest score or of 1: compared in 64 bits

struct RouteParams {
    const void *logits;
    const float *bias;                  // [experts] or null
    int64_t ld;
    int32_t *ids;
    float *weights;
    int32_t m, experts, top_k, score, dtype, renormalize;
    float scale;
};

// Larger floats have larger keys; 0 stands for what is never chosen.
__device__ __forceinline__ uint32_t route_order(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float route_unorder(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

__device__ __forceinline__ float route_score(float l, int kind) {
    if (kind == WS_SCORE_SIGMOID) return l >= 0.0f ? 1.0f / (1.0f + expf(-l)) : expf(l) / (1.0f + expf(l));
    return sqrtf(l > 0.0f ? l + log1pf(expf(-l)) : log1pf(expf(l)));
}
__device__ __forceinline__ double route_score64(double l, int kind) {
    if (kind == WS_SCORE_SIGMOID) return l >= 0.0 ? 1.0 / (1.0 + exp(-l)) : exp(l) / (1.0 + exp(l));
    return sqrt(l > 0.0 ? l + log1p(exp(-l)) : log1p(exp(l)));
}

// For the order alone, to 1e-6: exponential and logarithm as the hardware has them; small arguments of ln(1 + x), whose
// roots would show its absolute error, by its series.  (With the functions above 4096 tokens of 384 experts took 29 us.)
__device__ __forceinline__ float route_key(float l, int kind) {
    float x, y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(fabsf(l) * -1.4426950408889634f));     // e^-|l|
    if (kind == WS_SCORE_SIGMOID) {
        y = __fdividef(1.0f, 1.0f + x);
        return l >= 0.0f ? y : x * y;
    }
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(1.0f + x));
    const float series = x * fmaf(x, fmaf(x, fmaf(x, fmaf(x, 0.2f, -0.25f), 0.33333333f), -0.5f), 1.0f);
    y = x < 0.03125f ? series : y * 0.69314718f;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(l, 0.0f) + y));
    return y;
}

template <int N, bool F32>  // logits a lane
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const __grid_constant__ RouteParams p) {
    const int t = blockIdx.x * (kRouteThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    if (t >= p.m) return;
    const int64_t row = (int64_t)t * p.ld;
    const bool soft = p.score == WS_SCORE_SOFTMAX;
    // All loads at once: predicated, because behind branches the compiler waits for one before it issues the next.
    float l[N], b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = i * 32 + lane, ok = e < p.experts;
        uint32_t w = F32 ? 0xFF800000u : 0xFF80u, c = 0u;
        if constexpr (F32)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "+r"(w) : "l"(static_cast<const float *>(p.logits) + row + e), "r"(ok) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\t.reg .b16 h;\n\tmov.b16 h, 0xFF80;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.b16 h, [%1];\n\tmov.b32 %0, {0, h};\n\t}"
                         : "=r"(w) : "l"(static_cast<const uint16_t *>(p.logits) + row + e), "r"(ok) : "memory");
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "+r"(c) : "l"(p.bias + e), "r"((int)(ok && p.bias)) : "memory");
        l[i] = __uint_as_float(w);
        b[i] = __uint_as_float(c);
    }
    // softmax over all experts, where its values themselves count
    float top = -__builtin_huge_valf(), total = 1.0f;
    if (soft && (p.bias || !p.renormalize)) {
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, l[i]);     // (a NaN counts as nothing)
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) total += l[i] > -__builtin_huge_valf() ? expf(l[i] - top) : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    const float over = 1.0f / total;
    // No score is above this: sqrt(ln(1 + e^l)) <= sqrt(max(l, 0) + 1).
    float reach = 1.0f;
    if (p.bias && p.score == WS_SCORE_SQRTSOFTPLUS) {
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) big = fmaxf(big, l[i]);
        reach = sqrtf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big))) + 1.0f);
    }
    uint32_t key[N];
    bool fine = true;                   // no two neighbours of the order are too close
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float k = l[i];
        if (p.bias) k = (soft ? expf(l[i] - top) * over : route_key(l[i], p.score)) + b[i];
        key[i] = l[i] > -__builtin_huge_valf() && k == k ? route_order(k + 0.0f) : 0u;     // (+ 0: -0 and 0 are one)
    }
    // ---- rounds: the largest key left, of the lowest index
    int mine = -1;                      // lane j: the j-th expert
    float before = __builtin_huge_valf(), last = 0.0f;
    const int rounds = p.top_k + (p.bias ? 1 : 0);      // one more: how close the first that is left out comes
    // A softmax over a logit of +inf is NaN for all; with a bias the keys are, without one they are the logits.
    const uint32_t none = soft && !p.bias ? route_order(__builtin_huge_valf()) : 0u;
    uint32_t best = 0u;                 // of this lane's keys that are left
    uint32_t left[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        left[i] = key[i];
        best = max(best, key[i]);
    }
#pragma unroll 1
    for (int j = 0; j < rounds; ++j) {
        const uint32_t k = __reduce_max_sync(0xffffffffu, best);
        if (!k || k == none) break;
        int at = 0x7fffffff;            // its place, where this lane has it
        if (best == k) {
#pragma unroll
            for (int i = N - 1; i >= 0; --i) at = left[i] == k ? i * 32 + lane : at;
        }
        const int e = __reduce_min_sync(0xffffffffu, at);
        if (p.bias) {
            const float v = route_unorder(k);
            if (j && before - v <= kRouteNear * fmaxf(reach, fabsf(v))) fine = false;
            before = v;
        }
        if (j == p.top_k) break;
        last = before;
        if (lane == j) mine = e;
        if (at == e) {
            best = 0u;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                left[i] = i == e >> 5 ? 0u : left[i];
                best = max(best, left[i]);
            }
        }
    }
    if (p.bias && !fine) {              // (all lanes alike; rare, so the logits are read again)
        const float bound = last - kRouteNear * fmaxf(reach, fabsf(last));
        auto logit = [&](int i) { return i * 32 + lane < p.experts ? load1(p.logits, p.dtype, row + i * 32 + lane) : -__builtin_huge_valf(); };
        double total64 = 1.0;
        if (soft) {
            total64 = 0.0;
#pragma unroll 1
            for (int i = 0; i < N; ++i) {
                const float v = logit(i);
                total64 += v > -__builtin_huge_valf() ? exp((double)v - (double)top) : 0.0;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) total64 += __shfl_xor_sync(0xffffffffu, total64, o);
        }
        uint32_t close = 0u;            // this lane's candidates
#pragma unroll
        for (int i = 0; i < N; ++i) close |= key[i] && route_unorder(key[i]) >= bound ? 1u << i : 0u;
#pragma unroll 1
        for (int j = 0; j < p.top_k; ++j) {
            double bk = -__builtin_huge_val();
            int bi = -1;
            for (uint32_t left = close; left; left &= left - 1) {
                const int i = __ffs(left) - 1;
                const float v = logit(i);
                const double k = (soft ? exp((double)v - (double)top) / total64 : route_score64(v, p.score)) + (double)p.bias[i * 32 + lane];
                if (bi < 0 || k > bk) { bk = k; bi = i * 32 + lane; }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const double ok = __shfl_xor_sync(0xffffffffu, bk, o);
                const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
                if (oi >= 0 && (bi < 0 || ok > bk || (ok == bk && oi < bi))) { bk = ok; bi = oi; }
            }
            if (bi < 0) break;
            if ((bi & 31) == lane) close &= ~(1u << (bi >> 5));
            if (lane == j) mine = bi;
        }
    }
    // ---- weights
    const bool have = mine >= 0;
    const float mine_l = have ? load1(p.logits, p.dtype, row + mine) : 0.0f;
    float w = 0.0f, sum = 1.0f;
    if (soft) {
        float of = top;
        if (p.renormalize) {            // a ratio of the chosen: their own maximum will do
            of = have ? mine_l : -__builtin_huge_valf();
#pragma unroll
            for (int o = 16; o; o >>= 1) of = fmaxf(of, __shfl_xor_sync(0xffffffffu, of, o));
        } else {
            sum = total;
        }
        w = have ? expf(mine_l - of) : 0.0f;
    } else {
        w = have ? route_score(mine_l, p.score) : 0.0f;
    }
    if (p.renormalize) {
        sum = w;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!soft && sum < 1e-30f) {    // scores at the type's end: their ratios in 64 bits
            double w64 = have ? route_score64(mine_l, p.score) : 0.0, sum64 = w64;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum64 += __shfl_xor_sync(0xffffffffu, sum64, o);
            w = sum64 > 0.0 ? (float)(w64 / sum64) : 0.0f;
            sum = 1.0f;
        }
    }
    if (lane < p.top_k) {
        p.ids[(int64_t)t * p.top_k + lane] = mine;
        p.weights[(int64_t)t * p.top_k + lane] = have ? p.scale * (w / sum) : 0.0f;
    }
}

}  // namespace ws
