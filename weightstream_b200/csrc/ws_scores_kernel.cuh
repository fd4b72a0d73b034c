// Scores of given tokens on a row of logits: log probability, entropy, rank, and the best alternatives, from one pass.
//
// Every thread keeps the running maximum M of what it has seen with  s = sum exp(x - M)  and  t = sum exp(x - M) (x - M),
// both rescaled when M moves:  lse = M + ln s,  entropy = ln s - t / s.  A row is read by a cluster of 1 to 8 blocks,
// whose statistics meet in the first block's shared memory.
//
// The alternatives cost the pass nothing but the vector in which a thread's maximum lies: the k-th best of 64 groups'
// maxima is a lower bound of the k-th best value, and only threads whose maximum reaches it can hold an alternative.
// Their values (about k threads') are read once more, and what reaches the bound is ranked in shared memory.
//
// Order of values: larger first, equal ones by index, as argmax has it (crates/weightstream-ref/src/sample.rs:13-23).
// -inf (masked) and NaN are never alternatives.
#pragma once

#include <cooperative_groups.h>

#include "ws_norm_kernel.cuh"

namespace ws {

constexpr int kScoreThreads = 512;
constexpr int kScoreGroups = kScoreThreads / 8;   // groups of eight lanes whose maxima give the bound
constexpr int kScoreBatch = 4;                    // vectors a thread requests together
constexpr int kScoreMaxTop = 32;
constexpr int kScoreMaxCluster = 8;
constexpr float kLowest = -3.402823466e+38f, kNegInf = -__builtin_huge_valf();
constexpr float kFarBelow = -10000.0f;            // exp of it is 0 and its product with 0 is 0, as exp(-inf) (-inf) is not
static_assert(kScoreMaxTop <= kScoreGroups, "the bound needs a group for every alternative");

struct ScoreParams {
    const void *logits, *tokens;
    int64_t ld;
    int32_t m, vocab, top, token_bytes, cluster;
    float *logprob, *entropy, *top_logprob;
    int32_t *rank, *top_id;
};

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one of them is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// (value, index) as one number that is larger for what comes first; 0 is below all of them.  -0 and 0 are equal.
__device__ __forceinline__ uint64_t score_key(float v, uint32_t idx) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return ((uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int32_t key_index(uint64_t k) { return (int32_t)(0xFFFFFFFFu - (uint32_t)k); }

// A row as 16-byte vectors of its memory; the first and the last may lie partly outside, which reads as -inf.
template <bool F32>
struct ScoreRow {
    static constexpr int E = F32 ? 4 : 8;
    const char *base;      // 16-byte aligned, at most 15 bytes before the row
    int32_t lead, vocab;   // values of the first vector that lie before the row
    __device__ __forceinline__ ScoreRow(const void *p, int32_t v) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        base = reinterpret_cast<const char *>(a & ~(uintptr_t)15);
        lead = (int32_t)(a & 15) / (F32 ? 4 : 2);
        vocab = v;
    }
    __device__ __forceinline__ int32_t vectors() const { return (int32_t)(((int64_t)lead + vocab + E - 1) / E); }
    __device__ __forceinline__ int32_t first(int32_t v) const { return v * E - lead; }
    __device__ __forceinline__ uint4 raw(int32_t v) const {
        const int32_t i0 = first(v);
        if (i0 >= 0 && i0 <= vocab - E) return __ldg(reinterpret_cast<const uint4 *>(base) + v);
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (F32) {
                const int32_t i = i0 + j;
                w[j] = i >= 0 && i < vocab ? __ldg(reinterpret_cast<const uint32_t *>(base) + (int64_t)v * 4 + j) : 0xFF800000u;
            } else {
                const int32_t i = i0 + 2 * j;
                const uint16_t *q = reinterpret_cast<const uint16_t *>(base) + (int64_t)v * 8 + 2 * j;
                w[j] = (i >= 0 && i < vocab ? (uint32_t)__ldg(q) : 0xFF80u) |
                       (i + 1 >= 0 && i + 1 < vocab ? (uint32_t)__ldg(q + 1) << 16 : 0xFF800000u);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void values(const uint4 &r, float (&x)[E]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (F32) x[j] = __uint_as_float(w[j]);
            else {
                x[(2 * j) % E] = __uint_as_float(w[j] << 16);
                x[(2 * j + 1) % E] = __uint_as_float(w[j] & 0xFFFF0000u);
            }
        }
    }
};

struct ScoreStats {
    float m, s, t;
    int32_t before;
};
// Moves s and t to the maximum `to` >= m.
__device__ __forceinline__ void rebase(ScoreStats &a, float to) {
    const float d = fmaxf(a.m - to, kFarBelow), f = ex2f(d * 1.44269504f);
    a.t = f * fmaf(d, a.s, a.t);
    a.s *= f;
    a.m = to;
}

struct ScoreShared {
    uint64_t buf[kScoreThreads + kScoreThreads * 8];  // values that reach the bound: a round adds at most eight a thread
    uint64_t best[kScoreMaxTop];                      // this block's alternatives in order, 0 where there are no more
    uint64_t group[kScoreGroups];
    uint64_t bound;
    ScoreStats stats;                                 // this block's
    float warp_m[kScoreThreads / 32], warp_s[kScoreThreads / 32], warp_t[kScoreThreads / 32];
    int32_t warp_before[kScoreThreads / 32];
    int32_t list[kScoreThreads], listed, found;
};

// The `top` first of buf[0, n), n <= kScoreThreads, in order into best[]; the rest of best[] is 0.
__device__ __forceinline__ void rank_candidates(const uint64_t *buf, int n, int top, uint64_t *best) {
    const int tid = threadIdx.x;
    if (tid < top && tid >= n) best[tid] = 0;
    if (tid < n) {
        const uint64_t k = buf[tid];
        int r = 0;
        for (int j = 0; j < n; ++j) r += buf[j] > k || (buf[j] == k && j < tid);
        if (r < top) best[r] = k;
    }
    __syncthreads();
}

// Too many values reach the bound (many equal maxima, or few threads hold all large values): the `top` first of buf[0, n)
// by repeated maxima, back into buf[0, top).  The bound rises to the last of them.
__device__ __noinline__ void shrink_candidates(ScoreShared &sh, int n, int top) {
    const int tid = threadIdx.x, lane = tid & 31;
    uint64_t last = ~(uint64_t)0;
    for (int r = 0; r < top; ++r) {
        uint64_t k = 0;
        for (int i = tid; i < n; i += kScoreThreads) {
            const uint64_t c = sh.buf[i];
            if (c < last && c > k) k = c;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const uint64_t c = __shfl_xor_sync(0xffffffffu, k, o);
            if (c > k) k = c;
        }
        if (lane == 0) sh.group[tid >> 5] = k;
        __syncthreads();
        for (int w = 0; w < kScoreThreads / 32; ++w)
            if (sh.group[w] > k) k = sh.group[w];
        if (tid == 0) sh.best[r] = k;
        last = k;
        __syncthreads();
    }
    if (tid < top) sh.buf[tid] = sh.best[tid];
    if (tid == 0) {
        sh.found = top;
        sh.bound = last;
    }
    __syncthreads();
}

template <bool F32, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) token_scores_kernel(const __grid_constant__ ScoreParams p) {
    namespace cg = cooperative_groups;
    using Row = ScoreRow<F32>;
    constexpr int E = Row::E;
    __shared__ ScoreShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = blockIdx.x % p.cluster;
    const int64_t row = blockIdx.x / p.cluster;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    const Row x(static_cast<const char *>(p.logits) + row * p.ld * (F32 ? 4 : 2), p.vocab);
    const int64_t tok = p.token_bytes == 8 ? static_cast<const int64_t *>(p.tokens)[row] : static_cast<const int32_t *>(p.tokens)[row];
    const bool has_tok = tok >= 0 && tok < p.vocab;
    const float mine = has_tok ? load1(p.logits, F32 ? WS_ACT_F32 : WS_ACT_BF16, row * p.ld + tok) : __uint_as_float(0x7FC00000u);
    const int64_t all = x.vectors();
    const int32_t v0 = (int32_t)(all * part / p.cluster), v1 = (int32_t)(all * (part + 1) / p.cluster);

    ScoreStats a{kLowest, 0.0f, 0.0f, 0};
    float best = kNegInf;   // maximum of this thread's values, and the first vector that holds it
    int32_t best_v = 0;
    for (int32_t v = v0 + tid; v < v1; v += kScoreBatch * kScoreThreads) {
        uint4 raw[kScoreBatch];
#pragma unroll
        for (int j = 0; j < kScoreBatch; ++j) {
            const int32_t w = v + j * kScoreThreads;
            raw[j] = F32 ? make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u) : make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);
            if (w < v1) raw[j] = x.raw(w);
        }
        float most[kScoreBatch], big = kNegInf;
#pragma unroll
        for (int j = 0; j < kScoreBatch; ++j) {
            float c[E];
            Row::values(raw[j], c);
            most[j] = c[0];
#pragma unroll
            for (int e = 1; e < E; ++e) most[j] = fmaxf(most[j], c[e]);
            big = fmaxf(big, most[j]);
        }
        if (big > best) {
            best = big;
            rebase(a, big);
#pragma unroll
            for (int j = kScoreBatch - 1; j >= 0; --j)
                if (most[j] == big) best_v = v + j * kScoreThreads;
        }
#pragma unroll
        for (int j = 0; j < kScoreBatch; ++j) {
            float c[E];
            Row::values(raw[j], c);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = max_nan(c[e] - a.m, kFarBelow), q = ex2f(d * 1.44269504f);
                a.s += q;
                a.t = fmaf(q, d, a.t);
            }
        }
        if (big >= mine) {
            // the batch lies before the token, where equal values count, or behind it, or around it (or holds places
            // outside the row that look like a masked token)
            const int32_t i0 = x.first(v), i1 = x.first(v + (kScoreBatch - 1) * kScoreThreads) + E;
            const bool front = i1 <= tok && mine > kNegInf, behind = i0 > tok;
            if (front || behind) {
#pragma unroll
                for (int j = 0; j < kScoreBatch; ++j) {
                    float c[E];
                    Row::values(raw[j], c);
#pragma unroll
                    for (int e = 0; e < E; ++e) a.before += front ? c[e] >= mine : c[e] > mine;
                }
            } else {
#pragma unroll 1
                for (int j = 0; j < kScoreBatch; ++j) {
                    const int32_t w = v + j * kScoreThreads;
                    if (w >= v1) break;
                    float c[E];
                    Row::values(x.raw(w), c);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int32_t i = x.first(w) + e;
                        a.before += (c[e] > mine || (c[e] == mine && i < tok)) && i >= 0 && i < p.vocab;
                    }
                }
            }
        }
    }

    // the block's statistics
    float m = a.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    rebase(a, m);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
        a.before += __shfl_xor_sync(0xffffffffu, a.before, o);
    }
    if (lane == 0) {
        sh.warp_m[warp] = a.m;
        sh.warp_s[warp] = a.s;
        sh.warp_t[warp] = a.t;
        sh.warp_before[warp] = a.before;
    }
    uint64_t key = 0;
    if (TOP) {
        key = best > kNegInf ? score_key(best, (uint32_t)best_v) : 0;
        uint64_t g = key;
#pragma unroll
        for (int o = 4; o; o >>= 1) {
            const uint64_t c = __shfl_xor_sync(0xffffffffu, g, o);
            if (c > g) g = c;
        }
        if ((lane & 7) == 0) sh.group[tid >> 3] = g;
        if (tid == 0) sh.listed = sh.found = 0;
    }
    __syncthreads();
    if (warp == 0) {
        constexpr int W = kScoreThreads / 32;
        ScoreStats b{lane < W ? sh.warp_m[lane] : kLowest, lane < W ? sh.warp_s[lane] : 0.0f, lane < W ? sh.warp_t[lane] : 0.0f,
                     lane < W ? sh.warp_before[lane] : 0};
        float bm = b.m;
#pragma unroll
        for (int o = 16; o; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
        rebase(b, bm);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            b.s += __shfl_xor_sync(0xffffffffu, b.s, o);
            b.t += __shfl_xor_sync(0xffffffffu, b.t, o);
            b.before += __shfl_xor_sync(0xffffffffu, b.before, o);
        }
        if (lane == 0) sh.stats = b;
    }
    if (TOP) {
        // the top-th best of the groups' maxima: every group is compared with eight others by each of eight threads
        const int i = tid >> 3, j0 = (tid & 7) * (kScoreGroups / 8);
        const uint64_t g = sh.group[i];
        int r = 0;
#pragma unroll
        for (int j = j0; j < j0 + kScoreGroups / 8; ++j) r += sh.group[j] > g || (sh.group[j] == g && j < i);
#pragma unroll
        for (int o = 4; o; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
        // ... as a bound on single values: the last value of that vector
        if ((tid & 7) == 0 && r == p.top - 1) sh.bound = g == 0 ? 1 : (g & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (uint32_t)(x.first(key_index(g)) + E - 1));
        __syncthreads();
        uint64_t bound = sh.bound;
        // (this thread's best vector as a single value: its first, so that none of the vector is lost)
        if (key != 0 && ((key & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (uint32_t)max(x.first(best_v), 0))) >= bound) sh.list[atomicAdd(&sh.listed, 1)] = tid;
        __syncthreads();
        const int rounds = (v1 - v0 + kScoreThreads - 1) / kScoreThreads, items = sh.listed * rounds;
        for (int w0 = 0; w0 < items; w0 += kScoreThreads) {
            const int w = w0 + tid;
            if (w < items) {
                const int32_t v = v0 + sh.list[w / rounds] + (w % rounds) * kScoreThreads;
                if (v < v1) {
                    float c[E];
                    Row::values(x.raw(v), c);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (!(c[e] > kNegInf)) continue;
                        const uint64_t k = score_key(c[e], (uint32_t)(x.first(v) + e));
                        if (k >= bound) sh.buf[atomicAdd(&sh.found, 1)] = k;
                    }
                }
            }
            __syncthreads();
            if (sh.found > kScoreThreads) {
                shrink_candidates(sh, sh.found, p.top);
                bound = sh.bound;
            }
            __syncthreads();
        }
        rank_candidates(sh.buf, sh.found, p.top, sh.best);
    } else {
        __syncthreads();
    }

    // the row's
    ScoreStats b = sh.stats;
    if (p.cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (part == 0) {
            float bm = kLowest;
            for (int c = 0; c < p.cluster; ++c) bm = fmaxf(bm, cl.map_shared_rank(&sh, c)->stats.m);
            b = ScoreStats{bm, 0.0f, 0.0f, 0};
            for (int c = 0; c < p.cluster; ++c) {
                ScoreStats o = cl.map_shared_rank(&sh, c)->stats;
                rebase(o, bm);
                b.s += o.s;
                b.t += o.t;
                b.before += o.before;
            }
            if (TOP) {
                if (tid < p.cluster * p.top) sh.buf[tid] = cl.map_shared_rank(&sh, tid / p.top)->best[tid % p.top];
                __syncthreads();
            }
        }
        cl.sync();  // no block leaves while its shared memory is read
        if (part != 0) return;
        if (TOP) rank_candidates(sh.buf, p.cluster * p.top, p.top, sh.best);
    }
    const float ln_s = logf(b.s);
    if (tid == 0) {
        const bool none = b.s == 0.0f;
        const float h = ln_s - __fdividef(b.t, b.s);
        p.logprob[row] = !has_tok ? 0.0f : none ? kNegInf : (mine - b.m) - ln_s;
        p.entropy[row] = none ? 0.0f : h < 0.0f ? 0.0f : h;
        p.rank[row] = has_tok && mine == mine ? b.before : -1;
    }
    if (TOP && tid < p.top) {
        const uint64_t k = sh.best[tid];
        p.top_id[row * p.top + tid] = k ? key_index(k) : -1;
        p.top_logprob[row * p.top + tid] = k ? (key_value(k) - b.m) - ln_s : kNegInf;
    }
}

}  // namespace ws
