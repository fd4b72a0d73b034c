// Scores of given tokens on a row of logits: log probability, entropy, rank, and the best alternatives, from one pass.
//
// Every thread keeps  s = sum exp(x - M)  and  t = sum exp(x - M) (x - M)  for an M near the maximum of what it has seen
// (up to 16 below it: exp(16) times the values' count is far from the type's end), both rescaled when M moves:  lse = M + ln s,  entropy = ln s - t / s.  A row is read by a cluster of 1 to 8 blocks,
// which store their statistics and alternatives into the first block's shared memory.
//
// The alternatives cost the pass little: the k-th best of 64 groups' maxima is a lower bound of the k-th best value, and
// only threads whose maximum reaches it can hold an alternative.  After a sixteenth and a quarter of the row the bound is
// taken, and values that reach it are noted as they pass; at the end it is taken again, the first sixteenth's values of
// the threads whose maximum reaches it (about k threads) are read once more (a row that is one batch still has them in
// registers), and what is left is ranked in shared memory.
//
// Bound: HBM for fp32 rows (2000 rows of 129280: 167 us, 6.2 TB/s, in a graph of such calls 163 us), instructions for bf16
// ones (117 us, 4.4 TB/s: about ten a value, of which one is the exponential and two keep masked values from giving NaN) and
// for alternatives (twenty of them: 190 us and 187 us; five under a mask of 40 % of the vocabulary 204 us), latency for few
// rows (one row with twenty alternatives 10 us and without 6, 64 rows with twenty 18 us and without 10).
//
// Order of values: larger first, equal ones by index, as argmax has it (crates/weightstream-ref/src/sample.rs:13-23).
// -inf (masked) and NaN are never alternatives.
#pragma once

#include <cooperative_groups.h>

#include "ws_norm_kernel.cuh"

namespace ws {

constexpr int kScoreGroups = 64;                  // groups of neighbouring threads whose maxima give the bound
constexpr int kScoreBatch = 4;                    // vectors a thread works on together
constexpr int kScoreMaxTop = 32;
template <int T, bool F32>
constexpr int kScoreRings = T == 512 || F32 ? 2 : 3;  // batches in flight and at work
constexpr int kScoreMaxCluster = 8;
constexpr float kLowest = -3.402823466e+38f, kNegInf = -__builtin_huge_valf();
constexpr float kScoreSlack = 16.0f;
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
__device__ __forceinline__ float warp_max(float v) {  // on all lanes; NaN counts as nothing
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// Two floats at a time: the sums of a pass are issue-bound otherwise.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float one_gt(float a, float b) {  // 1 where it holds, else 0
    float r;
    asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float one_ge(float a, float b) {
    float r;
    asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void async_copy16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

constexpr int kScoreNoted = 1024;                     // values noted in passing; more: all are read once more
template <int T>
struct ScoreShared {
    // values that reach the bound: up to T wait while a round of reading adds at most eight a thread
    alignas(16) uint64_t buf[T + T * 8];
    uint64_t best[T];                                 // in the first block: every block's alternatives in order, 0 where there are no more
    uint64_t group[kScoreGroups];
    uint64_t bound;
    ScoreStats warp[kScoreMaxCluster * T / 32];       // in the first block: those of the cluster's warps
    int32_t list[T], listed, found, kept;
};

// The `top` first of the distinct keys buf[0, n), n <= T, in order into best[]; the rest of best[] is 0.
template <int T>
__device__ __forceinline__ void rank_candidates(const uint64_t *buf, int n, int top, uint64_t *best) {
    const int tid = threadIdx.x;
    int g = 1;  // threads to a key
    while (g < 32 && n * g * 2 <= T) g *= 2;
    const int i = tid / g;
    int r = 0;
    const uint64_t k = i < n ? buf[i] : 0;
    if (i < n) {
#pragma unroll 4
        for (int j = tid % g; j < n; j += g) r += buf[j] > k;
    }
    for (int o = g / 2; o; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    if (i < n && tid % g == 0 && r < top) best[r] = k;
    if (tid >= n && tid < top) best[tid] = 0;
}

// Too many values reach the bound (many equal maxima, or few threads hold all large values): the `top` first of buf[0, n)
// by repeated maxima, back into buf[0, top).  The bound rises to the last of them.
template <int T>
__device__ __noinline__ void shrink_candidates(ScoreShared<T> &sh, int n, int top) {
    const int tid = threadIdx.x, lane = tid & 31;
    uint64_t last = ~(uint64_t)0, mine = 0;  // (thread r keeps the r-th)
    for (int r = 0; r < top; ++r) {
        uint64_t k = 0;
        for (int i = tid; i < n; i += T) {
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
        for (int w = 0; w < T / 32; ++w)
            if (sh.group[w] > k) k = sh.group[w];
        if (tid == r) mine = k;
        last = k;
        __syncthreads();
    }
    if (tid < top) sh.buf[tid] = mine;
    if (tid == 0) {
        sh.found = top;
        sh.bound = last;
    }
    __syncthreads();
}

// Bound of single values: the top-th best of the groups' maxima, given as (value, batch) of every thread, and of that
// batch its last value.
template <int T, typename F>
__device__ __forceinline__ uint64_t take_bound(ScoreShared<T> &sh, const F &last_of, uint64_t key, int top) {
    constexpr int G = T / kScoreGroups;   // threads of a group
    const int tid = threadIdx.x;
#pragma unroll
    for (int o = G / 2; o; o >>= 1) {
        const uint64_t c = __shfl_xor_sync(0xffffffffu, key, o);
        if (c > key) key = c;
    }
    if (tid % G == 0) sh.group[tid / G] = key;
    __syncthreads();
    // every group is compared with all, a part of them by each of its threads
    const int i = tid / G, j0 = tid % G * (kScoreGroups / G);
    const uint64_t g = sh.group[i];
    int r = 0;
#pragma unroll
    for (int j = j0; j < j0 + kScoreGroups / G; ++j) r += sh.group[j] > g || (sh.group[j] == g && j < i);
#pragma unroll
    for (int o = G / 2; o; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    if (tid % G == 0 && r == top - 1) sh.bound = g == 0 ? 1 : (g & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (uint32_t)last_of(key_index(g)));
    __syncthreads();
    return sh.bound;
}

template <int T, bool F32>
constexpr int kScoreSmem = sizeof(ScoreShared<T>) + kScoreRings<T, F32> * kScoreBatch * T * 16;

template <int T, bool F32, bool TOP>
__global__ void __launch_bounds__(T, T == 512 ? 2 : F32 ? 4 : 3) token_scores_kernel(const __grid_constant__ ScoreParams p) {
    namespace cg = cooperative_groups;
    using Row = ScoreRow<F32>;
    constexpr int E = Row::E, kBatch = kScoreBatch, kStep = kBatch * T;
    constexpr int kScoreRing = kScoreRings<T, F32>;
    constexpr uint32_t kMasked = F32 ? 0xFF800000u : 0xFF80FF80u;
    extern __shared__ __align__(16) uint8_t score_smem[];
    ScoreShared<T> &sh = *reinterpret_cast<ScoreShared<T> *>(score_smem);
    uint4 *const ring = reinterpret_cast<uint4 *>(score_smem + sizeof(ScoreShared<T>));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = blockIdx.x % p.cluster;
    const int64_t row = blockIdx.x / p.cluster;
    cg::cluster_group cl = cg::this_cluster();
    if (p.cluster > 1) cl.barrier_arrive();  // waited for before the first block's shared memory is written
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    const Row x(static_cast<const char *>(p.logits) + row * p.ld * (F32 ? 4 : 2), p.vocab);
    const int64_t all = x.vectors();
    const int32_t v0 = (int32_t)(all * part / p.cluster), v1 = (int32_t)(all * (part + 1) / p.cluster);
    // Batches are requested a ring's length ahead, straight into shared memory; a thread reads back what it asked for.
    const int batches = (v1 - v0 + kStep - 1) / kStep;   // the same for all threads of the block
    auto vector = [&](int b, int j) { return v0 + b * kStep + j * T + tid; };
    // batches [inner0, inner1) hold nothing but whole vectors of the row
    const int inner0 = x.first(v0) < 0 ? 1 : 0, inner1 = (min(v1, (p.vocab + x.lead) / E) - v0) / kStep;
    int slot_in = 0, slot_out = 0;   // places of the ring
    const char *ahead = x.base + ((int64_t)v0 + tid) * 16;
    auto request = [&](int b) {
        uint4 *slot = ring + slot_in * kStep + tid;
        if (b >= inner0 && b < inner1) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) async_copy16(slot + j * T, ahead + j * T * 16);
        } else if (b < batches) {
#pragma unroll 1
            for (int j = 0; j < kBatch; ++j) {
                const int32_t v = vector(b, j);
                slot[j * T] = v < v1 ? x.raw(v) : make_uint4(kMasked, kMasked, kMasked, kMasked);
            }
        }
        async_commit();
        ahead += kStep * 16;
        slot_in = slot_in + 1 == kScoreRing ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int b = 0; b + 1 < kScoreRing; ++b) request(b);
    const int64_t tok = p.token_bytes == 8 ? static_cast<const int64_t *>(p.tokens)[row] : static_cast<const int32_t *>(p.tokens)[row];
    const bool has_tok = tok >= 0 && tok < p.vocab;
    const float mine = has_tok ? load1(p.logits, F32 ? WS_ACT_F32 : WS_ACT_BF16, row * p.ld + tok) : __uint_as_float(0x7FC00000u);

    auto last_of = [&](int b) { return x.first(min(v0 + (b + 1) * kStep, v1)) - 1; };
    const int early = TOP && batches > 2 ? (batches + 15) / 16 : batches, later = 4 * early;
    if (TOP && tid == 0) sh.listed = sh.found = sh.kept = 0;
    float m = kLowest, best = kNegInf;   // m: what s and t refer to; best: maximum of this thread's values
    int32_t best_b = 0, before = 0;      // the first batch that holds it
    float2 s2 = make_float2(0.0f, 0.0f), t2 = s2, many = s2;  // many: counts of at most 2^23, a thread's share of a row
    float note = __uint_as_float(0x7FC00000u);  // values from here on are noted; NaN: none
    uint4 raw[kBatch];
    for (int b = 0; b < batches; ++b) {
        if (TOP && (b == early || b == later)) {
            const uint64_t k = take_bound(sh, last_of, best > kNegInf ? score_key(best, (uint32_t)best_b) : 0, p.top);
            note = k == 1 ? kNegInf : key_value(k);  // 1: too few groups hold anything yet, so all that follows counts
        }
        const int32_t v = vector(b, 0);
        request(b + kScoreRing - 1);
        async_wait<kScoreRing - 1>();
#pragma unroll
        for (int j = 0; j < kBatch; ++j) raw[j] = ring[slot_out * kStep + j * T + tid];
        const uint4 *const here = ring + slot_out * kStep + tid;
        slot_out = slot_out + 1 == kScoreRing ? 0 : slot_out + 1;
        float most[kBatch], big = kNegInf;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            float c[E];
            Row::values(raw[j], c);
            most[j] = c[0];
#pragma unroll
            for (int e = 1; e < E; ++e) most[j] = fmaxf(most[j], c[e]);
            big = fmaxf(big, most[j]);
        }
        if (big > best) {
            best = big;
            best_b = b;
        }
        if (big > m + kScoreSlack) {
            const float d = fmaxf(m - big, kFarBelow), f = ex2f(d * 1.44269504f);
            const float2 d2 = make_float2(d, d), f2 = make_float2(f, f);
            t2 = mul2(f2, fma2(d2, s2, t2));
            s2 = mul2(f2, s2);
            m = big;
        }
        const float2 m2 = make_float2(-m, -m);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            float c[E];
            Row::values(raw[j], c);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float2 d = add2(make_float2(c[e], c[e + 1]), m2);
                d.x = max_nan(d.x, kFarBelow);
                d.y = max_nan(d.y, kFarBelow);
                float2 q = mul2(d, make_float2(1.44269504f, 1.44269504f));
                q.x = ex2f(q.x);
                q.y = ex2f(q.y);
                s2 = add2(s2, q);
                t2 = fma2(q, d, t2);
            }
        }
        if (big >= mine) {
            // the batch lies before the token, where equal values count, or behind it, or around it (or holds places
            // outside the row that look like a masked token)
            const int32_t i0 = x.first(v), i1 = x.first(v + (kBatch - 1) * T) + E;
            if (i0 > tok) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    float c[E];
                    Row::values(raw[j], c);
#pragma unroll
                    for (int e = 0; e < E; e += 2) many = add2(many, make_float2(one_gt(c[e], mine), one_gt(c[e + 1], mine)));
                }
            } else if (i1 <= tok && mine > kNegInf) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    float c[E];
                    Row::values(raw[j], c);
#pragma unroll
                    for (int e = 0; e < E; e += 2) many = add2(many, make_float2(one_ge(c[e], mine), one_ge(c[e + 1], mine)));
                }
            } else {
#pragma unroll 1
                for (int j = 0; j < kBatch; ++j) {
                    const int32_t w = v + j * T;
                    if (w >= v1) break;
                    float c[E];
                    Row::values(x.raw(w), c);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int32_t i = x.first(w) + e;
                        before += (c[e] > mine || (c[e] == mine && i < tok)) && i >= 0 && i < p.vocab;
                    }
                }
            }
        }
        if (TOP && big >= note) {
            // (nearly half of a warp's batches hold such a value, almost always one: the vector that does is looked at where it
            // lies, in a loop, which keeps this code small)
            uint32_t hits = 0;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) hits |= (most[j] >= note ? 1u : 0u) << j;
#pragma unroll 1
            for (; hits; hits &= hits - 1) {
                const int j = __ffs(hits) - 1;
                float c[E];
                Row::values(here[j * T], c);
                const int32_t i0 = x.first(v + j * T);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (c[e] >= note && c[e] > kNegInf) {
                        const int at = atomicAdd(&sh.found, 1);
                        if (at < kScoreNoted) sh.buf[at] = score_key(c[e], (uint32_t)(i0 + e));
                    }
            }
        }
    }
    ScoreStats a{m, s2.x + s2.y, t2.x + t2.y, before + (int32_t)many.x + (int32_t)many.y};

    // the warps' statistics, into the first block
    ScoreShared<T> *const first = p.cluster > 1 ? cl.map_shared_rank(&sh, 0) : &sh;
    rebase(a, fmaxf(warp_max(best), kLowest));
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    a.before = __reduce_add_sync(0xffffffffu, a.before);
    if (p.cluster > 1) cl.barrier_wait();
    if (lane == 0) first->warp[part * (T / 32) + warp] = a;
    if (TOP) {
        const uint64_t key = best > kNegInf ? score_key(best, (uint32_t)best_b) : 0;
        uint64_t bound = take_bound(sh, last_of, key, p.top);
        // threads whose best batch (by its first value, so that none of it is lost) reaches the bound
        const bool reaches = key != 0 && ((key & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (uint32_t)max(x.first(v0 + best_b * kStep), 0))) >= bound;
        if (batches == 1) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                if (reaches) {
                    float c[E];
                    Row::values(raw[j], c);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint64_t k = score_key(c[e], (uint32_t)(x.first(vector(0, j)) + e));
                        if (c[e] > kNegInf && k >= bound) sh.buf[atomicAdd(&sh.found, 1)] = k;
                    }
                }
                __syncthreads();
                if (sh.found > T) {
                    shrink_candidates(sh, sh.found, p.top);
                    bound = sh.bound;
                }
                __syncthreads();
            }
        } else {
            // of what was noted, what reaches the bound now
            const int noted = sh.found;
            const bool again = noted > kScoreNoted;  // not all of it is there
            if (reaches) sh.list[atomicAdd(&sh.listed, 1)] = tid;
            if (noted && !again) {
                uint64_t keep[kScoreNoted / T];
#pragma unroll
                for (int i = 0; i < kScoreNoted / T; ++i) keep[i] = tid + i * T < noted ? sh.buf[tid + i * T] : 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kScoreNoted / T; ++i)
                    if (keep[i] >= bound) sh.buf[atomicAdd(&sh.kept, 1)] = keep[i];
            }
            __syncthreads();
            const int rounds = (again ? batches : early) * kBatch, items = sh.listed * rounds;
            if (tid == 0) sh.found = sh.kept;
            __syncthreads();
            for (int w0 = 0;; w0 += T) {
                if (sh.found > T) {
                    shrink_candidates(sh, sh.found, p.top);
                    bound = sh.bound;
                }
                __syncthreads();
                if (w0 >= items) break;
                const int w = w0 + tid;
                if (w < items) {
                    const int32_t v = v0 + sh.list[w / rounds] + (w % rounds) * T;
                    if (v < v1) {
                        float c[E];
                        Row::values(x.raw(v), c);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const uint64_t k = score_key(c[e], (uint32_t)(x.first(v) + e));
                            if (c[e] > kNegInf && k >= bound) sh.buf[atomicAdd(&sh.found, 1)] = k;
                        }
                    }
                }
                __syncthreads();
            }
        }
        rank_candidates<T>(sh.buf, sh.found, p.top, first->best + part * p.top);
    }

    // the row's
    if (p.cluster > 1) cl.sync();
    else __syncthreads();
    if (part != 0) return;
    if (TOP && p.cluster > 1) {
        // the best of the blocks' last ones is a bound again
        uint64_t bound = 1;
        for (int c = 0; c < p.cluster; ++c) {
            const uint64_t k = sh.best[c * p.top + p.top - 1];
            if (k > bound) bound = k;
        }
        const uint64_t k = tid < p.cluster * p.top ? sh.best[tid] : 0;
        if (tid == 0) sh.found = 0;
        __syncthreads();
        if (k >= bound) sh.buf[atomicAdd(&sh.found, 1)] = k;
        __syncthreads();
        rank_candidates<T>(sh.buf, sh.found, p.top, sh.best);
        __syncthreads();
    }
    if (warp != 0) return;
    ScoreStats b{kLowest, 0.0f, 0.0f, 0};
    const int warps = p.cluster * (T / 32);
    for (int w = lane; w < warps; w += 32) b.m = fmaxf(b.m, sh.warp[w].m);
    b.m = warp_max(b.m);
    for (int w = lane; w < warps; w += 32) {
        ScoreStats o = sh.warp[w];
        rebase(o, b.m);
        b.s += o.s;
        b.t += o.t;
        b.before += o.before;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        b.s += __shfl_xor_sync(0xffffffffu, b.s, o);
        b.t += __shfl_xor_sync(0xffffffffu, b.t, o);
    }
    b.before = __reduce_add_sync(0xffffffffu, b.before);
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
