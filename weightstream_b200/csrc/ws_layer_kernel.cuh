// A whole mixture-of-experts layer of a few tokens over MXFP4 experts, in two kernels and a sum:
//
//   first    g = W1[e] x,  u = W3[e] x,  h = weight * silu(g) * u        (clamped first, where a limit is given)
//   second   y[t] = sum over t's routes of W2[e] h
//
// Every weight byte is used by the few tokens that chose its expert, so the layer is bound by HBM.  Weights stream
// through rings in shared memory that each warp keeps for itself (asynchronous copies, no barriers between warps), are
// widened to f16 (exact) and multiplied by mma.sync with the tokens as its 8 columns.  The order of a contraction's
// terms is free: a lane takes 8 consecutive codes of a row, one word, as the terms that the instruction's layout gives
// it.  A scale holds for 32 codes of a row, so two products of 16 terms are added up in the tensor core and then, times
// the scale, in fp32.
//
// Activations are f16 too, without loss of theirs: a token's row is scaled by the power of two that brings its largest
// value below 2^15, so a bf16 value is held exactly down to 2^-29 of the largest and to 2^-40 of it absolutely; fp32
// values take two columns, a value and what its rounding to f16 left, together 22 bits or more down to 2^-17 of the
// largest and 2^-40 of it absolutely.  With act_quant the rows are first rounded as the steps' quantiser does.
//
// A pass is one expert with as many of its routes as the columns hold, a unit a tile of 16 weight rows of a pass (first
// kernel: 8 of W1 and the same 8 of W3, so that a lane has both of a value's products) or two of W2.  Every block takes a
// contiguous share of all passes' units; its warps, in groups that share K, take them in turn.
//
// The second kernel's results of a route go to a workspace, and a third, small launch adds up a token's routes in the order
// of its slots.  (Who brings the last of a token's routes adding them up in the second kernel took 40 to 90 us more with 48
// to 96 routes: popular experts' blocks ended late.)
//
// Bound: HBM, and what stands before the streams.  One token of 7168 x 2048 through six experts 43 us, of which HBM needs 21:
// routes, plan and activations 8, W1 and W3 17 (5.6 TB/s), the second kernel's beginning 7, W2 9 (5.1 TB/s), the sum 2.  48
// routes of 30 experts 165 to 173 us (107), 96 of 42 233 to 241 us (150), fp32 activations rounded to E4M3, 28 routes of 20 experts of 5120
// x 2304, 103 to 106 us (57).  At HBM's rate the issue slots, the conversions of codes and shared memory are each half to three
// quarters busy: 30 instructions a lane for 16 codes, of which 8 convert, 2 multiply and 4 add.
//
// mma.sync and not tcgen05: its block-scaled form takes activations of 8 bits at most, so that a bf16 value held exactly
// would be two columns and an fp32 value six, and sums over all of K are cut at every step there; the tensor pipe is a
// quarter busy here.
#pragma once

#include <type_traits>

#include "ws_values.cuh"

namespace ws {

constexpr int kLayerWarps = 12;
constexpr int kLayerThreads = kLayerWarps * 32;
constexpr int kLayerBlocks = 148;
constexpr int kLayerMaxRoutes = 512, kLayerMaxExperts = 512, kLayerMaxTopK = 8;    // as the routed step's
constexpr int kLayerMaxWidth = 24576;
constexpr int kLayerChunk = 256;                    // values of K a stage: 128 bytes of 16 rows
constexpr int kLayerPitch = 144;                    // (rows 16 bytes beyond their data: a warp's words lie in all banks)
constexpr int kLayerScales = 16 * kLayerPitch;      // where a stage's scales begin: 8 bytes of 16 rows, or the three words that hold them
template <bool FULL>
constexpr int kLayerStage = kLayerScales + 16 * (FULL ? 8 : 12);
constexpr int kLayerMaxPasses = 16;                 // of a block's share: at most 512 / 148 + 2
static_assert(kLayerMaxRoutes / kLayerBlocks + 3 <= kLayerMaxPasses, "a block's passes");

struct LayerParams {
    const void *x;                                  // first: [m, k] activations
    const int32_t *ids;                             // [m, top_k] global experts
    const float *weights;                           // [m, top_k]
    const uint8_t *wa, *sa, *wb, *sb;               // first: W1, W3 and their scales; second: W2 twice
    int64_t ldx, wa_e, sa_e, wb_e, sb_e, ldo;       // strides: of x and out in elements, of experts in bytes
    float *h;                                       // [m * top_k, rows of W1]
    float *part;                                    // [m * top_k, rows of W2] results of the routes
    void *out;
    int32_t x_dtype, out_dtype, m, top_k, e_start, e_len, act_quant, has_limit;
    int32_t k, units;                               // contraction, units a pass
    int32_t n;                                      // width of the result: of h, of part and out
    int32_t per, room;                              // routes a pass; rows of activations that shared memory holds
    int32_t vec;                                    // x is read 16 bytes at a time (the sum: out is written so)
    float limit;
};

__device__ __forceinline__ void layer_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a block adds to zeros that stay in registers: as constants the compiler makes them anew each time.
__device__ __forceinline__ void layer_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&zero)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(zero[0]), "f"(zero[1]), "f"(zero[2]), "f"(zero[3]));
}
__device__ __forceinline__ void layer_copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void layer_copy8(uint32_t dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void layer_copy4(uint32_t dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void layer_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void layer_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Eight values of a column, where there is one.
__device__ __forceinline__ void layer_column(uint4 &v, uint32_t at, bool have) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "r"(at), "r"((int)have));
}
// Byte B of a scale word as 2^(b - 127); 0 gives 0 (2^-127, below what a sum of normal numbers holds), 255 infinity.
template <int B>
__device__ __forceinline__ float layer_scale(uint32_t w) { return __uint_as_float((B == 3 ? w >> 1 : w << (23 - 8 * B)) & 0x7F800000u); }
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16_lo(uint32_t v) {
    float r;
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.f32.f16 %0, l;}" : "=f"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float f16_hi(uint32_t v) {
    float r;
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.f32.f16 %0, h;}" : "=f"(r) : "r"(v));
    return r;
}
// Eight values of a row; what the kernel before this one wrote is not read through the read-only path.
__device__ __forceinline__ void layer_load8(const void *p, int dtype, bool vec, int64_t i, bool ok, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (!ok) return;
    if (!vec) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = load1(p, dtype, i + e);
    } else if (dtype == WS_ACT_F32) {
        const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
        const float4 a = __ldcg(q), b = __ldcg(q + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 r = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(w[e] << 16);
            v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
        }
    }
}
__host__ __device__ constexpr int layer_column_pitch(int k) { return 2 * k + (k % 64 ? 0 : 64); }  // 64 bytes past a multiple of 128: two columns' words lie in all banks

// What a block knows of the batch: routes of every expert, the passes of its share and their routes.
struct LayerPlan {
    int16_t ids[kLayerMaxRoutes];                   // local expert of a route, -1: none here
    int32_t first[kLayerMaxExperts];                // an expert's routes
    int32_t expert[kLayerMaxPasses], routes[kLayerMaxPasses], start[kLayerMaxPasses + 1];   // start: a pass' first entry of `route`
    int16_t route[kLayerMaxPasses * 8];
    int32_t pass0, pass1, passes;                   // of the share
    int32_t unit0, unit1;                           // the share, counted from its first pass' first unit
    int64_t warp_sum[kLayerWarps];
    int32_t group;                                  // warps that share a unit
    int32_t scale[kLayerMaxPasses * 8];             // of the routes' rows, as powers of two
    uint32_t amax[kLayerMaxPasses * 8];
};

// What a unit of a pass of n routes costs, in fortieths: an SM's part of HBM while the columns' loads and products are hidden
// by it (24 experts of 7168 x 2048, all with n routes, n = 1, 4, 8: first kernel 66, 68, 73 us; second 35, 36, 53).  With one cost
// for all: 96 routes of 48 experts of 7168 x 2048 211 us instead of 197, 256 routes of 32 of 1024 x 512 39 instead of 33, others within 6 %.
template <bool FIRST>
__device__ __forceinline__ int layer_cost(const LayerParams &p, int n) { return FIRST ? 40 + n / 2 : n <= 4 ? 40 : 57; }

// Warps that share a unit by K, for units of this cost together: the more, the less the warps wait for the last one at the
// end; the fewer, the less often they join their sums.  One warp a unit everywhere, us: 12 routes of 24 experts of 7168 x 2048 66 instead
// of 63, 128 routes of 64 of 7168 x 256 71 instead of 67; but 128 routes of 32 of 4096 x 1536 88 instead of 100, 32 routes of 64 of 1024 x
// 512 21 instead of 24, so the rule is not the best one for all widths.  Four everywhere: slower throughout, 140 instead of 89 with 512
// routes of 128 of 2048 x 768.
template <bool FIRST>
__device__ __forceinline__ int layer_group(const LayerParams &p, int64_t all) {
    const int chunks = (p.k + kLayerChunk - 1) / kLayerChunk, each = (int)(all / gridDim.x) / layer_cost<FIRST>(p, 1);    // units a block
    // (short rows, many units: a call of 48 routes of 30 experts 166 us with a unit a warp in the second kernel, 170 with two warps)
    const int group = chunks >= 16 ? 4 : chunks >= 4 && each < 3 * kLayerWarps ? 2 : 1;
    return each < kLayerWarps / group ? 4 : group;
}

template <bool FIRST>
__device__ __forceinline__ void layer_plan(LayerPlan &s, const LayerParams &p) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, routes = p.m * p.top_k, per = p.per;
    if (routes <= 32) {
        // A route a lane, all of it in one warp: an expert's routes are lanes that match, its first lane stands for it, and
        // experts are put in order by comparing the first lanes.  (An expert with more than a pass of routes takes the way below.)
        if (tid < kLayerMaxPasses * 8) s.amax[tid] = 0u;
        if (warp == 0) {
            const int64_t wide = lane < routes ? (int64_t)p.ids[lane] - p.e_start : -1;
            const int e = lane < routes && p.ids[lane] >= 0 && wide >= 0 && wide < p.e_len ? (int)wide : -1;
            if (lane < routes) s.ids[lane] = (int16_t)e;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const int n = __popc(same), cost = layer_cost<FIRST>(p, n);
            const bool first = e >= 0 && (same & ((1u << lane) - 1u)) == 0u;
            const bool many = __any_sync(0xffffffffu, e >= 0 && n > per);
            int pass = 0, cheaper = 0, total = 0, start = 0;    // passes, cost and routes of the experts before this one
#pragma unroll 4
            for (int l = 0; l < routes; ++l) {
                const int other = __shfl_sync(0xffffffffu, first ? e : -1, l), c = __shfl_sync(0xffffffffu, cost, l), k = __shfl_sync(0xffffffffu, n, l);
                if (other < 0) continue;
                total += c;
                if (other < e) {
                    ++pass;
                    cheaper += c;
                    start += k;
                }
            }
            const int64_t all = (int64_t)total * p.units, x0 = all * blockIdx.x / gridDim.x, x1 = all * (blockIdx.x + 1) / gridDim.x;
            const int64_t from = (int64_t)cheaper * p.units, to = from + (int64_t)cost * p.units;
            const bool mine = first && to > x0 && from < x1 && x1 > x0;
            const uint32_t all_mine = __ballot_sync(0xffffffffu, mine);
            const int pass0 = __reduce_min_sync(0xffffffffu, mine ? pass : 0x7fffffff), start0 = __reduce_min_sync(0xffffffffu, mine ? start : 0x7fffffff);
            const int passes = __popc(all_mine);
            if (mine) {
                const int i = pass - pass0;
                s.expert[i] = e;
                s.routes[i] = n;
                s.start[i] = start - start0;
                if (from <= x0) s.unit0 = (int)((x0 - from + cost - 1) / cost);
                if (to >= x1) {
                    s.unit1 = (int)min((int64_t)p.units, (x1 - from + cost - 1) / cost) + i * p.units;
                    s.start[passes] = start - start0 + n;
                }
            }
            const bool routed = __shfl_sync(0xffffffffu, (int)mine, __ffs(same) - 1);
            if (e >= 0 && routed) s.route[start - start0 + __popc(same & ((1u << lane) - 1u))] = (int16_t)lane;
            if (lane == 0) {
                s.passes = many ? -1 : passes;
                if (!passes) s.unit0 = s.unit1 = 0;
                s.group = layer_group<FIRST>(p, all);
            }
        }
        __syncthreads();
        if (s.passes >= 0) return;
        __syncthreads();
    }
    int32_t id[(kLayerMaxRoutes + kLayerThreads - 1) / kLayerThreads];
#pragma unroll
    for (int i = 0; i < (kLayerMaxRoutes + kLayerThreads - 1) / kLayerThreads; ++i) id[i] = i * kLayerThreads + tid < routes ? p.ids[i * kLayerThreads + tid] : -1;
    for (int i = tid; i < p.e_len; i += kLayerThreads) s.first[i] = 0;
    if (tid < kLayerMaxPasses * 8) s.amax[tid] = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (kLayerMaxRoutes + kLayerThreads - 1) / kLayerThreads; ++i) {
        const int64_t e = (int64_t)id[i] - p.e_start;
        const bool ok = id[i] >= 0 && e >= 0 && e < p.e_len;
        if (i * kLayerThreads + tid < routes) s.ids[i * kLayerThreads + tid] = ok ? (int16_t)e : (int16_t)-1;
        if (ok) atomicAdd(&s.first[(int)e], 1);
    }
    __syncthreads();
    // Passes of every expert, added up, and what their units cost: a thread takes neighbouring experts.
    const int each = (p.e_len + kLayerThreads - 1) / kLayerThreads, e0 = tid * each, e1 = min(p.e_len, e0 + each);
    int64_t mine = 0;                               // cost << 16 | passes
    for (int e = e0; e < e1; ++e) {
        const int n = s.first[e], full = n / per, rest = n - full * per;
        mine += ((int64_t)(full * layer_cost<FIRST>(p, per) + (rest ? layer_cost<FIRST>(p, rest) : 0)) << 16) + full + (rest ? 1 : 0);
    }
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) s.warp_sum[warp] = before;
    if (tid == 0) s.passes = 0;
    __syncthreads();
    int64_t at = before - mine, total = 0;
#pragma unroll 1
    for (int w = 0; w < kLayerWarps; ++w) {
        if (w < warp) at += s.warp_sum[w];
        total += s.warp_sum[w];
    }
    // The block's share of all cost, [x0, x1): the units that begin in it.
    const int64_t all = (total >> 16) * p.units, x0 = all * blockIdx.x / gridDim.x, x1 = all * (blockIdx.x + 1) / gridDim.x;
    int64_t from = (at >> 16) * p.units;            // where the thread's first pass begins
    int pass = (int)(at & 0xFFFF);
#pragma unroll 1
    for (int e = e0; e < e1; ++e) {
        const int n = s.first[e];
#pragma unroll 1
        for (int skip = 0; skip < n; skip += per, ++pass) {
            const int here = min(per, n - skip), cost = layer_cost<FIRST>(p, here);
            const int64_t to = from + (int64_t)cost * p.units;
            if (to > x0 && from < x1) {
                // the block's first pass is the one that x0 lies in, and places count from it
                if (from <= x0) {
                    s.pass0 = pass;
                    s.unit0 = (int)((x0 - from + cost - 1) / cost);
                }
                if (to >= x1) {
                    s.pass1 = pass;
                    s.unit1 = (int)min((int64_t)p.units, (x1 - from + cost - 1) / cost);
                }
                const int i = pass & (kLayerMaxPasses - 1);     // (a share has fewer passes than places)
                s.expert[i] = e;
                s.routes[i] = here | skip << 16;
            }
            from = to;
        }
    }
    __syncthreads();
    const int pass0 = s.pass0, passes = x1 > x0 ? s.pass1 - pass0 + 1 : 0;
    int own = 0, own_routes = 0;
    if (tid < passes) {                             // places in order
        own = s.expert[(pass0 + tid) & (kLayerMaxPasses - 1)];
        own_routes = s.routes[(pass0 + tid) & (kLayerMaxPasses - 1)];
    }
    __syncthreads();
    if (tid < passes) {
        s.expert[tid] = own;
        s.routes[tid] = own_routes;
    }
    if (tid == 0) {
        s.passes = passes;
        s.unit1 = passes ? s.unit1 + (passes - 1) * p.units : 0;
        if (!passes) s.unit0 = 0;
        s.group = layer_group<FIRST>(p, all);
    }
    __syncthreads();
    for (int q = warp; q < passes; q += kLayerWarps) {  // the pass's routes, in their order
        int start = 0;
        for (int i = 0; i < q; ++i) start += s.routes[i] & 0xFFFF;
        const int e = s.expert[q], skip = s.routes[q] >> 16, n = s.routes[q] & 0xFFFF;
        int seen = 0;
        for (int i = 0; i < routes && seen < skip + n; i += 32) {
            const bool hit = i + lane < routes && s.ids[i + lane] == e;
            const uint32_t hits = __ballot_sync(0xffffffffu, hit);
            const int place = seen + __popc(hits & ((1u << lane) - 1u)) - skip;
            if (hit && place >= 0 && place < n) s.route[start + place] = (int16_t)(i + lane);
            seen += __popc(hits);
        }
        if (lane == 0) {
            s.start[q] = start;
            if (q == passes - 1) s.start[passes] = start + n;
        }
    }
    __syncthreads();
}

// Eight activations as f16, scaled; PAIR: what that rounds off too.
template <bool PAIR>
__device__ __forceinline__ void layer_put(const float (&v)[8], float scale, uint32_t at, uint32_t at_rest) {
    uint32_t a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x0 = v[2 * i] * scale, x1 = v[2 * i + 1] * scale;
        a[i] = f16x2(x0, x1);
        if constexpr (PAIR) {
            const float r0 = x0 - f16_lo(a[i]), r1 = x1 - f16_hi(a[i]);
            b[i] = f16x2(fabsf(x0) < 65536.0f ? r0 : 0.0f, fabsf(x1) < 65536.0f ? r1 : 0.0f);   // (an infinity has no remainder)
        }
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]) : "memory");
    if constexpr (PAIR) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at_rest), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3]) : "memory");
}
__device__ __forceinline__ uint32_t layer_larger(uint32_t big, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        big = b < 0x7F800000u ? max(big, b) : big;      // (infinities and NaN stay what they are)
    }
    return big;
}
// Eight values rounded as the steps' quantiser does; four neighbouring lanes hold a block of 32.
__device__ __forceinline__ void layer_round(float (&v)[8]) {
    int e;
    uint32_t lo, hi;
    act_quant8(v, e, lo, hi);
    const uint32_t w[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
    const float up = pow2_f32(e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = f16_lo(w[i]) * up;
        v[2 * i + 1] = f16_hi(w[i]) * up;
    }
}

// The columns of some passes: rows of activations as f16, scaled.  PAIR: two columns a row, value and remainder.  A row's
// values come to the place of their columns as they are, by asynchronous copies, and are turned there by the lane that
// copied them; rows that 16 bytes do not divide, and fp32 ones that get one column, are loaded twice instead.
// All rows' pieces of 256 values are dealt out to the warps in turn.
template <bool FIRST, bool PAIR>
struct LayerColumns {
    const LayerParams &p;
    uint32_t smem, pitch;
    int r0, pieces, each;                               // pieces of a row; of all rows

    __device__ __forceinline__ LayerColumns(const LayerParams &p, uint32_t smem, int r0, int n)
        : p(p), smem(smem), pitch(layer_column_pitch(p.k)), r0(r0), pieces((p.k + 255) / 256 * n), each((p.k + 255) / 256) {}
    __device__ __forceinline__ bool copied() const { return FIRST ? p.vec && PAIR == (p.x_dtype == WS_ACT_F32) : true; }
    __device__ __forceinline__ uint32_t place(int i) const { return smem + (uint32_t)(PAIR ? 2 * i : i) * pitch; }
    __device__ __forceinline__ int64_t row(const LayerPlan &s, int i) const { return FIRST ? s.route[r0 + i] / p.top_k * p.ldx : (int64_t)s.route[r0 + i] * p.k; }
    // f(rows, this lane's eight values of them) for the warp's pieces, N of them at once; whole warps.  Row -1: no piece.
    template <int N, typename F>
    __device__ __forceinline__ void deal(F f) const {
        int i = 0, c = threadIdx.x >> 5;                // of row i, piece c
#pragma unroll 1
        for (int q = c; q < pieces; q += N * kLayerWarps) {
            int rows[N], at[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                while (c >= each) {
                    c -= each;
                    ++i;
                }
                const int at8 = c * 32 + (int)(threadIdx.x & 31);
                rows[k] = q + k * kLayerWarps < pieces && at8 * 8 < p.k ? i : -1;
                at[k] = at8;
                c += kLayerWarps;
            }
            f(rows, at);
        }
    }
    __device__ __forceinline__ void request(const LayerPlan &s) const {
        if (copied())
            deal<1>([&](const int (&rows)[1], const int (&at)[1]) {
                const int i = rows[0], c = at[0];
                if (i < 0) return;
                const uint32_t to = place(i) + c * 16;
                const int64_t from = row(s, i) + c * 8;
                if constexpr (PAIR) {
                    const float *x = (FIRST ? static_cast<const float *>(p.x) : p.h) + from;
                    layer_copy16(to, x);
                    layer_copy16(to + pitch, x + 4);
                } else {
                    layer_copy16(to, static_cast<const uint16_t *>(p.x) + from);
                }
            });
        layer_commit();
    }
    __device__ __forceinline__ void value(const LayerPlan &s, int i, int c, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        if (i < 0) return;
        if (copied()) {
            const uint32_t at = place(i) + c * 16;
            const uint4 a = lds_u128(at);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
            if constexpr (PAIR) {
                const uint4 b = lds_u128(at + pitch);
                const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = __uint_as_float(w[e]);
                    v[4 + e] = __uint_as_float(u[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[2 * e] = __uint_as_float(w[e] << 16);
                    v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
                }
            }
        } else {
            layer_load8(p.x, p.x_dtype, p.vec, row(s, i) + c * 8, true, v);
        }
    }
    // The largest of eight values as they were copied, as the bits of an fp32 number; infinities and NaN among them.
    __device__ __forceinline__ uint32_t largest(int i, int c) const {
        if (i < 0) return 0u;
        const uint4 a = lds_u128(place(i) + c * 16);
        if constexpr (PAIR) {
            const uint4 b = lds_u128(place(i) + c * 16 + pitch);
            const uint32_t m = max(max(max(a.x & 0x7FFFFFFFu, a.y & 0x7FFFFFFFu), max(a.z & 0x7FFFFFFFu, a.w & 0x7FFFFFFFu)),
                                   max(max(b.x & 0x7FFFFFFFu, b.y & 0x7FFFFFFFu), max(b.z & 0x7FFFFFFFu, b.w & 0x7FFFFFFFu)));
            return m;
        } else {
            const uint32_t m = __vmaxu2(__vmaxu2(a.x & 0x7FFF7FFFu, a.y & 0x7FFF7FFFu), __vmaxu2(a.z & 0x7FFF7FFFu, a.w & 0x7FFF7FFFu));
            return max(m << 16, m & 0xFFFF0000u);
        }
    }
    // After the copies have come.
    __device__ __forceinline__ void turn(LayerPlan &s) const {
        deal<4>([&](const int (&rows)[4], const int (&at)[4]) {
            uint32_t big[4];
            if (copied()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) big[k] = largest(rows[k], at[k]);
            }
            if (!copied() || __any_sync(0xffffffffu, max(max(big[0], big[1]), max(big[2], big[3])) >= 0x7F800000u)) {
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    float v[8];
                    value(s, k == 0 ? rows[0] : k == 1 ? rows[1] : k == 2 ? rows[2] : rows[3], k == 0 ? at[0] : k == 1 ? at[1] : k == 2 ? at[2] : at[3], v);
                    const uint32_t m = layer_larger(0u, v);
                    big[0] = k == 0 ? m : big[0];
                    big[1] = k == 1 ? m : big[1];
                    big[2] = k == 2 ? m : big[2];
                    big[3] = k == 3 ? m : big[3];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) big[k] = __reduce_max_sync(0xffffffffu, big[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if ((threadIdx.x & 31) == 0 && rows[k] >= 0) atomicMax(&s.amax[r0 + rows[k]], big[k]);
        });
        __syncthreads();
        deal<4>([&](const int (&rows)[4], const int (&at)[4]) {
            float v[4][8];
#pragma unroll
            for (int k = 0; k < 4; ++k) value(s, rows[k], at[k], v[k]);
            if (p.act_quant)
#pragma unroll
                for (int k = 0; k < 4; ++k) layer_round(v[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = rows[k], c = at[k];
                if (i < 0) continue;
                // 2^-e brings the largest below 2^15 (rows below 2^-100 are scaled as if they reached it)
                const int e = max((int)(s.amax[r0 + i] >> 23) - 127, -100) - 14;
                if (c == 0) s.scale[r0 + i] = e;
                layer_put<PAIR>(v[k], pow2_f32(-e), place(i) + c * 16, place(i) + pitch + c * 16);
            }
        });
        __syncthreads();
    }
};

// Where a warp's copies are: the next chunk of K of a tile, as this lane copies it.  Eight lanes copy a row's 128 bytes (two
// lanes a row, with one address for all of a lane's copies, took 55 us instead of 45 for one token: the lines that an
// instruction touches are what it costs).
struct LayerSource {
    const uint8_t *a0, *a1, *b0, *b1;               // 16 bytes of rows r, r + 4, r + 8 and r + 12
    const uint8_t *s;                               // of scales
    int unit, tile, chunk;
};

// A block of 32 values of K of a tile, a word of codes of rows g and g + 8: products with CT tiles of columns, times the
// rows' scales.
template <int CT>
__device__ __forceinline__ void layer_block(float (&sum)[CT][4], uint4 (&x)[CT], uint32_t a, uint32_t b, const uint32_t (&col)[CT], const bool (&have)[CT], float s0, float s1,
                                            const float (&zero)[4]) {
    const uint32_t a0 = e2m1x2_byte_to_f16x2<0>(a), a1 = e2m1x2_byte_to_f16x2<1>(a), a2 = e2m1x2_byte_to_f16x2<2>(a), a3 = e2m1x2_byte_to_f16x2<3>(a);
    const uint32_t b0 = e2m1x2_byte_to_f16x2<0>(b), b1 = e2m1x2_byte_to_f16x2<1>(b), b2 = e2m1x2_byte_to_f16x2<2>(b), b3 = e2m1x2_byte_to_f16x2<3>(b);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        layer_column(x[t], col[t], have[t]);
        float d[4];
        layer_mma0(d, a0, b0, a1, b1, x[t].x, x[t].y, zero);
        layer_mma(d, a2, b2, a3, b3, x[t].z, x[t].w);
        sum[t][0] = fmaf(d[0], s0, sum[t][0]);
        sum[t][1] = fmaf(d[1], s0, sum[t][1]);
        sum[t][2] = fmaf(d[2], s1, sum[t][2]);
        sum[t][3] = fmaf(d[3], s1, sum[t][3]);
    }
}

// NT: most tiles of 8 columns, D stages a warp; FULL: K is whole chunks.
template <bool FIRST, bool PAIR, bool FULL, int NT, int D>
__global__ void __launch_bounds__(kLayerThreads, 1) layer_kernel(const __grid_constant__ LayerParams p) {
    constexpr int kStage = kLayerStage<FULL>, kTiles = FIRST ? 1 : 2;     // tiles of 16 rows a unit
    extern __shared__ __align__(128) uint8_t layer_smem[];
    __shared__ LayerPlan s;
    __shared__ __align__(16) float scale_s[kLayerWarps][16][8];           // a stage's scales
    const int tid = threadIdx.x, lane = tid & 31, warp = warp_id(), g = lane >> 2, tq = lane & 3;
    const int column = layer_column_pitch(p.k);
    const uint32_t ring = smem_u32(layer_smem) + warp * D * kStage, cols = smem_u32(layer_smem) + kLayerWarps * D * kStage;
    float *const red = reinterpret_cast<float *>(layer_smem + kLayerWarps * D * kStage + p.room * column * (PAIR ? 2 : 1));   // [2][warps][NT * 4][32]
    if constexpr (FIRST) {
        wait_predecessor();
        // The second kernel may begin: it reads the routes and the weights, which this wait has seen complete, before it
        // waits for this one.
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    layer_plan<FIRST>(s, p);
    const int chunks = (p.k + kLayerChunk - 1) / kLayerChunk, group = s.group, slice = warp % group, step = kLayerWarps / group;
    const int64_t kw = p.k / 2, ks = p.k / 32;
    // passes whose columns fit together
    auto batch = [&](int q) {
        int e = q + 1;
        while (e < s.passes && s.start[e + 1] - s.start[q] <= p.room) ++e;
        return e;
    };
    int q0 = 0, q1 = s.passes ? batch(0) : 0;
    if constexpr (FIRST)
        if (q1) LayerColumns<FIRST, PAIR>(p, cols, 0, s.start[q1]).request(s);
    // a tile's rows: FIRST 8 of W1 and the same of W3, else 16 of W2
    auto row_a = [&](int u, int tile) { return (int64_t)(FIRST ? u * 8 : u * 32 + tile * 16); };
    auto row_b = [&](int u, int tile) { return (int64_t)(FIRST ? u * 8 : u * 32 + tile * 16 + 8); };
    LayerSource src;
    src.unit = s.unit0 + warp / group;
    src.tile = 0;
    src.chunk = slice;
    const int unit1 = s.unit1, row = lane >> 3, part = lane & 7;     // of the copies: rows row, row + 4, ...; 16 bytes a part
    const int srow = lane >> 1, half = lane & 1;    // of the scales: 4 bytes of a row a lane
    const uint32_t put = ring + row * kLayerPitch + part * 16, sput = ring + kLayerScales + srow * (FULL ? 8 : 12) + half * 4;
    auto seek = [&]() {                             // the rows of src.unit
        const int q = src.unit / p.units, u = src.unit - q * p.units;
        const int64_t e = s.expert[q], ra = row_a(u, src.tile), rb = row_b(u, src.tile);
        src.a0 = p.wa + e * p.wa_e + (ra + row) * kw + src.chunk * (kLayerChunk / 2) + part * 16;
        src.b0 = p.wb + e * p.wb_e + (rb + row) * kw + src.chunk * (kLayerChunk / 2) + part * 16;
        src.a1 = src.a0 + 4 * kw;
        src.b1 = src.b0 + 4 * kw;
        src.s = (srow < 8 ? p.sa + e * p.sa_e + (ra + srow) * ks : p.sb + e * p.sb_e + (rb + srow - 8) * ks) + src.chunk * (kLayerChunk / 32);
    };
    if (slice >= chunks) src.unit = unit1;          // (a short K has no share for this warp)
    if (src.unit < unit1) seek();
    // Copies the next chunk to a stage; a warp without one commits an empty group, so that groups count stages.
    auto request = [&](int stage) {
        if (src.unit < unit1) {
            const uint32_t at = put + stage * kStage, sat = sput + stage * kStage;
            const int blocks = FULL ? 8 : min(kLayerChunk / 32, (p.k - src.chunk * kLayerChunk) / 32);
            if (FULL || part < blocks) {
                layer_copy16(at, src.a0);
                layer_copy16(at + 4 * kLayerPitch, src.a1);
                layer_copy16(at + 8 * kLayerPitch, src.b0);
                layer_copy16(at + 12 * kLayerPitch, src.b1);
            }
            if constexpr (FULL) {
                layer_copy4(sat, src.s + half * 4);
            } else {
                // the words that a row's scales lie in: up to three, the third by the first lane
                const uintptr_t from = reinterpret_cast<uintptr_t>(src.s) & ~(uintptr_t)3;
                const int end = (int)(reinterpret_cast<uintptr_t>(src.s) & 3) + blocks;
                if (half * 4 < end) layer_copy4(sat, reinterpret_cast<const void *>(from + half * 4));
                if (!half && end > 8) layer_copy4(sat + 8, reinterpret_cast<const void *>(from + 8));
            }
            const int ahead = group * (kLayerChunk / 2);
            src.chunk += group;
            src.a0 += ahead;
            src.a1 += ahead;
            src.b0 += ahead;
            src.b1 += ahead;
            src.s += group * (kLayerChunk / 32);
            if (src.chunk >= chunks) {
                src.chunk = slice;
                if (kTiles == 1 || ++src.tile == kTiles) {
                    src.tile = 0;
                    src.unit += step;
                }
                if (src.unit < unit1) seek();
            }
        }
        layer_commit();
    };
#pragma unroll 1
    for (int i = 0; i < D - 1; ++i) request(i);
    if constexpr (!FIRST) {
        wait_predecessor();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        if (q1) LayerColumns<FIRST, PAIR>(p, cols, 0, s.start[q1]).request(s);
    }
    const uint32_t decoded = smem_u32(scale_s[warp]);
    float zero[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("mov.f32 %0, 0f00000000;" : "=f"(zero[i]));
    int unit = s.unit0 + warp / group, stage = 0, flip = 0;
    // A tile's sums over this warp's share of K.
    auto tile_sums = [&](auto ct, float (&sum)[NT][4], int q, int u, int tile, int r0, int n) {
        constexpr int CT = decltype(ct)::value;
        float part_sum[CT][4];
        // This lane's columns.  Lanes whose column no route has never load: their values stay zero.
        uint32_t col[CT];
        bool have[CT];
        uint4 x[4][CT];                             // of four blocks of 32, so that loads run ahead
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            have[t] = t * 8 + g < (PAIR ? 2 * n : n);
            col[t] = cols + (uint32_t)(((PAIR ? 2 * r0 : r0) + t * 8 + g) * column) + tq * 16 + slice * (kLayerChunk * 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j][t] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < 4; ++i) part_sum[t][i] = 0.0f;
        }
        for (int chunk = slice; chunk < chunks; chunk += group) {
            layer_wait<D - 2>();
            __syncwarp();                           // all of this stage has come, and the one before it is free
            request(stage == 0 ? D - 1 : stage - 1);
            const uint32_t at = ring + stage * kStage, words = at + (lane & 15) * kLayerPitch + (lane >> 4) * 16;
            // The rows' scales in fp32, four by each lane: every lane needs those of rows g and g + 8.
            {
                const int r = lane >> 1, h = lane & 1;
                uint32_t w;
                if constexpr (FULL) {
                    w = lds_u32(at + kLayerScales + r * 8 + h * 4);
                } else {
                    const int64_t e = s.expert[q];
                    const uint8_t *from = r < 8 ? p.sa + e * p.sa_e + (row_a(u, tile) + r) * ks : p.sb + e * p.sb_e + (row_b(u, tile) + r - 8) * ks;
                    const int shift = (int)(reinterpret_cast<uintptr_t>(from + chunk * 8) & 3) * 8;
                    w = __funnelshift_r(lds_u32(at + kLayerScales + r * 12 + h * 4), lds_u32(at + kLayerScales + r * 12 + h * 4 + 4), shift);
                }
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(decoded + r * 32 + h * 16), "f"(layer_scale<0>(w)), "f"(layer_scale<1>(w)), "f"(layer_scale<2>(w)),
                             "f"(layer_scale<3>(w)) : "memory");
                __syncwarp();
            }
            const int blocks = FULL ? 8 : min(8, (p.k - chunk * kLayerChunk) / 32);
            if (FULL || blocks == 8) {
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    const uint4 sa = lds_u128(decoded + g * 32 + j * 4), sb = lds_u128(decoded + (g + 8) * 32 + j * 4);
                    const uint32_t fa[4] = {sa.x, sa.y, sa.z, sa.w}, fb[4] = {sb.x, sb.y, sb.z, sb.w};
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        uint32_t w[4];              // words of rows g and g + 8 of two blocks
                        ldmatrix_x4(words + (j + i) * 16, w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t c[CT];
#pragma unroll
                            for (int t = 0; t < CT; ++t) c[t] = col[t] + (j + i + h) * 64;
                            layer_block<CT>(part_sum, x[i + h], w[2 * h], w[2 * h + 1], c, have, __uint_as_float(fa[i + h]), __uint_as_float(fb[i + h]), zero);
                        }
                    }
                }
            } else {
                for (int j = 0; j < blocks; ++j) {
                    uint32_t c[CT];
#pragma unroll
                    for (int t = 0; t < CT; ++t) c[t] = col[t] + j * 64;
                    const uint32_t own = at + g * kLayerPitch + tq * 4 + j * 16;
                    layer_block<CT>(part_sum, x[0], lds_u32(own), lds_u32(own + 8 * kLayerPitch), c, have, lds_f32(decoded + g * 32 + j * 4), lds_f32(decoded + (g + 8) * 32 + j * 4), zero);
                }
            }
#pragma unroll
            for (int t = 0; t < CT; ++t) col[t] += group * (kLayerChunk * 2);
            stage = stage == D - 1 ? 0 : stage + 1;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[t][i] = t < CT ? part_sum[t < CT ? t : 0][i] : 0.0f;
    };
    while (q1) {
        {
            const LayerColumns<FIRST, PAIR> columns(p, cols, s.start[q0], s.start[q1] - s.start[q0]);
            if (q0) {
                __syncthreads();                    // the batch before this one has been read
                columns.request(s);
            }
            if (FIRST && !q0) layer_wait<D - 1>();  // (the weights' requests came after it)
            else layer_wait<0>();
            columns.turn(s);
        }
        const int end = min(s.unit1, q1 * p.units);
        for (; unit < end; unit += step) {
            const int q = unit / p.units, u = unit - q * p.units, start = s.start[q], n = s.routes[q] & 0xFFFF;
#pragma unroll 1
            for (int tile = 0; tile < kTiles; ++tile) {
                float sum[NT][4];
                if (NT > 1 && (PAIR ? 2 * n : n) > 8) tile_sums(std::integral_constant<int, NT>{}, sum, q, u, tile, start - s.start[q0], n);
                else tile_sums(std::integral_constant<int, 1>{}, sum, q, u, tile, start - s.start[q0], n);
                if (group > 1) {
                    // Shares of K, in the order of the warps.  (Two buffers take turns: who writes one again has met the
                    // first warp after that had read it.)
                    float *const mine = red + ((flip * kLayerWarps + warp) * NT * 4) * 32 + lane;
                    if (slice)
#pragma unroll
                        for (int i = 0; i < NT * 4; ++i) mine[i * 32] = sum[i / 4][i % 4];
                    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / group), "r"(group * 32) : "memory");
                    flip ^= 1;
                    if (slice) continue;
                    for (int w = 1; w < group; ++w)
#pragma unroll
                        for (int i = 0; i < NT * 4; ++i) sum[i / 4][i % 4] += mine[(w * NT * 4 + i) * 32];
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int i = 0; i < (PAIR ? 1 : 2); ++i) {
                        const int r = PAIR ? j * 4 + tq : j * 8 + tq * 2 + i;
                        if (r >= n) continue;
                        const int route = s.route[start + r];
                        const float up2 = pow2_f32(s.scale[start + r]);
                        const float va = (PAIR ? sum[j][0] + sum[j][1] : sum[j][i]) * up2, vb = (PAIR ? sum[j][2] + sum[j][3] : sum[j][2 + i]) * up2;
                        if constexpr (FIRST) {
                            float gate = va, up = vb;
                            if (p.has_limit) {
                                gate = gate > p.limit ? p.limit : gate;                 // (a NaN stays one)
                                up = up > p.limit ? p.limit : up < -p.limit ? -p.limit : up;
                            }
                            p.h[(int64_t)route * p.n + u * 8 + g] = p.weights[route] * (gate / (1.0f + expf(-gate)) * up);
                        } else {
                            float *const to = p.part + (int64_t)route * p.n + u * 32 + tile * 16 + g;
                            to[0] = va;
                            to[8] = vb;
                        }
                    }
                }
            }
        }
        q0 = q1;
        q1 = q0 < s.passes ? batch(q0) : 0;
    }
    layer_wait<0>();
}

// A token's routes on this rank, added up in the order of its slots.
constexpr int kLayerSumThreads = 128;
__global__ void __launch_bounds__(kLayerSumThreads) layer_sum_kernel(const __grid_constant__ LayerParams p) {
    const int per_row = p.n / 4, i = blockIdx.x * kLayerSumThreads + threadIdx.x, t = i / per_row, c = (i - t * per_row) * 4;
    wait_predecessor();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (t >= p.m) return;
    const int32_t *const ids = p.ids + t * p.top_k;
    const float *const from = p.part + (int64_t)t * p.top_k * p.n + c;
    float4 v[kLayerMaxTopK];
#pragma unroll
    for (int j = 0; j < kLayerMaxTopK; ++j) {
        const int64_t e = j < p.top_k ? (int64_t)ids[j] - p.e_start : -1;
        v[j] = e >= 0 && e < p.e_len && ids[j] >= 0 ? __ldcg(reinterpret_cast<const float4 *>(from + (int64_t)j * p.n)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float4 y = v[0];
#pragma unroll
    for (int j = 1; j < kLayerMaxTopK; ++j) {
        y.x += v[j].x;
        y.y += v[j].y;
        y.z += v[j].z;
        y.w += v[j].w;
    }
    const float o[4] = {y.x, y.y, y.z, y.w};
    if (p.vec) {                                    // (of out here)
        if (p.out_dtype == WS_ACT_F32) *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + t * p.ldo + c) = y;
        else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + t * p.ldo + c) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) store1(p.out, p.out_dtype, t * p.ldo + c + e, o[e]);
    }
}

}  // namespace ws
