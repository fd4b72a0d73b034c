// A whole mixture-of-experts layer of a few tokens over MXFP4 experts, in two kernels:
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
// kernel: 8 of W1 and the same 8 of W3, so that a lane has both of a value's products).  Every block takes a contiguous
// share of all passes' units; its warps (few units: groups of two or four warps that share K) take them in turn.
//
// The second kernel's results of a route go to a workspace, and the warp that brings the last of a token's routes to a
// tile adds them up in the order of the token's slots: the sums' order does not depend on who is last.
#pragma once

#include "ws_values.cuh"

namespace ws {

constexpr int kLayerWarps = 12;
constexpr int kLayerThreads = kLayerWarps * 32;
constexpr int kLayerBlocks = 148;
constexpr int kLayerMaxRoutes = 512, kLayerMaxExperts = 512, kLayerMaxTopK = 8;    // as the routed step's
constexpr int kLayerMaxWidth = 24576;
constexpr int kLayerChunk = 256;                    // values of K a stage: 128 bytes of 16 rows
constexpr int kLayerPitch = 144;                    // (rows 16 bytes beyond their data: a warp's words lie in all banks)
constexpr int kLayerStage = 16 * kLayerPitch + 16 * 12;
constexpr int kLayerMaxPasses = 16;                 // of a block's share: at most 512 / 148 + 2
static_assert(kLayerMaxRoutes / kLayerBlocks + 3 <= kLayerMaxPasses, "a block's passes");

struct LayerParams {
    const void *x;                                  // first: [m, k] activations
    const int32_t *ids;                             // [m, top_k] global experts
    const float *weights;                           // [m, top_k]
    const uint8_t *wa, *sa, *wb, *sb;               // first: W1, W3 and their scales; second: W2 twice
    int64_t ldx, wa_e, sa_e, wb_e, sb_e, ldo;       // strides: of x and out in elements, of experts in bytes
    float *h;                                       // [m * top_k, rows of W1]
    float *part;                                    // [m * top_k, n] results of the routes
    uint32_t *count;                                // [n / 16, m] routes that have come
    void *out;
    int32_t x_dtype, out_dtype, m, top_k, e_start, e_len, act_quant, has_limit;
    int32_t k, units;                               // contraction, units a pass
    int32_t n;                                      // second: width of out; first: tiles of the second, whose counts are cleared
    int32_t per;                                    // routes a pass
    int32_t vec;                                    // x is read 16 bytes at a time
    float limit;
};

__device__ __forceinline__ void layer_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void layer_copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void layer_copy4(uint32_t dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void layer_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void layer_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

// What a block knows of the batch: routes of every expert, and the passes of its share.
struct LayerPlan {
    int32_t ids[kLayerMaxRoutes];                   // local expert of a route, -1: none here
    int32_t first[kLayerMaxExperts + 1];            // an expert's first pass
    int32_t expert[kLayerMaxPasses], routes[kLayerMaxPasses];
    int16_t route[kLayerMaxPasses][8];
    uint8_t here[kLayerMaxRoutes];                  // a token's routes on this rank
    int32_t pass0, passes;                          // the share's first pass and how many
    int32_t unit0, unit1;                           // the share, counted from pass0's first unit
    int32_t warp_sum[kLayerWarps];
    int32_t group;                                  // warps that share a unit
    int32_t scale[8];                               // of the rows, as powers of two
    uint32_t amax[8];
    float red[kLayerWarps][8][32];                  // partial sums of warps that share a unit
};

__device__ __forceinline__ void layer_plan(LayerPlan &s, const LayerParams &p) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, routes = p.m * p.top_k, per = p.per;
    for (int i = tid; i < p.e_len; i += kLayerThreads) s.first[i] = 0;
    for (int i = tid; i < p.m; i += kLayerThreads) {
        int n = 0;
        for (int j = 0; j < p.top_k; ++j) {
            const int e = p.ids[i * p.top_k + j] - p.e_start;
            const bool ok = e >= 0 && e < p.e_len;
            s.ids[i * p.top_k + j] = ok ? e : -1;
            n += ok;
        }
        s.here[i] = (uint8_t)n;
    }
    __syncthreads();
    for (int i = tid; i < routes; i += kLayerThreads)
        if (s.ids[i] >= 0) atomicAdd(&s.first[s.ids[i]], 1);
    __syncthreads();
    // passes of every expert, added up: a thread takes neighbouring experts
    const int each = (p.e_len + kLayerThreads - 1) / kLayerThreads, e0 = tid * each, e1 = min(p.e_len, e0 + each);
    int mine = 0;
    for (int e = e0; e < e1; ++e) mine += (s.first[e] + per - 1) / per;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) s.warp_sum[warp] = before;
    __syncthreads();
    int at = before - mine, total = 0;
    for (int w = 0; w < kLayerWarps; ++w) {
        if (w < warp) at += s.warp_sum[w];
        total += s.warp_sum[w];
    }
    const int64_t units = (int64_t)total * p.units;
    const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
    const int pass0 = (int)(u0 / p.units), passes = u1 > u0 ? (int)((u1 - 1) / p.units) - pass0 + 1 : 0;
    if (tid == 0) {
        s.pass0 = pass0;
        s.passes = passes;
        s.unit0 = (int)(u0 - (int64_t)pass0 * p.units);
        s.unit1 = (int)(u1 - (int64_t)pass0 * p.units);
        // few units: more warps a unit, so that all of them have copies in flight
        const int64_t share = units / gridDim.x;
        s.group = share >= 8 ? 1 : share >= 4 ? 2 : 4;
    }
    for (int e = e0; e < e1; ++e) {                 // (counts give way to first passes)
        const int n = s.first[e], np = (n + per - 1) / per;
        for (int q = max(at, pass0); q < min(at + np, pass0 + passes); ++q) {
            s.expert[q - pass0] = e;
            s.routes[q - pass0] = min(per, n - (q - at) * per) | (q - at) * per << 16;
        }
        at += np;
    }
    __syncthreads();
    for (int q = warp; q < passes; q += kLayerWarps) {  // the pass's routes, in their order
        const int e = s.expert[q], skip = s.routes[q] >> 16, n = s.routes[q] & 0xFFFF;
        int seen = 0;
        for (int i = 0; i < routes && seen < skip + n; i += 32) {
            const bool hit = i + lane < routes && s.ids[i + lane] == e;
            const uint32_t hits = __ballot_sync(0xffffffffu, hit);
            const int place = seen + __popc(hits & ((1u << lane) - 1u)) - skip;
            if (hit && place >= 0 && place < n) s.route[q][place] = (int16_t)(i + lane);
            seen += __popc(hits);
        }
        __syncwarp();
        if (lane == 0) s.routes[q] = n;
    }
    __syncthreads();
}

// The columns of a pass: rows of activations as f16, scaled.  PAIR: two columns a row, value and remainder.
template <bool PAIR>
__device__ __forceinline__ void layer_columns(LayerPlan &s, const LayerParams &p, int q, bool first, uint32_t smem) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = s.routes[q], each = kLayerWarps / n < 1 ? 1 : kLayerWarps / n;
    const void *base = first ? p.x : p.h;
    const int dtype = first ? p.x_dtype : WS_ACT_F32;
    const int64_t ld = first ? p.ldx : p.k;
    const bool vec = !first || p.vec;
    if (tid < 8) s.amax[tid] = 0u;
    __syncthreads();
    const int col = warp / each, sub = warp % each;    // `each` warps a row
    const int64_t row = col < n ? (int64_t)(first ? s.route[q][col] / p.top_k : s.route[q][col]) * ld : 0;
    const int chunks = p.k / 8;
    if (col < n) {
        uint32_t big = 0u;
        for (int c = sub * 32 + lane; c < chunks; c += each * 32) {
            float v[8];
            layer_load8(base, dtype, vec, row + c * 8, true, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
                big = b < 0x7F800000u ? max(big, b) : big;      // (infinities and NaN stay what they are)
            }
        }
        big = __reduce_max_sync(0xffffffffu, big);
        if (lane == 0) atomicMax(&s.amax[col], big);
    }
    __syncthreads();
    if (col < n) {
        // 2^-e brings the largest below 2^15 (rows below 2^-100 are scaled as if they reached it)
        const int e = max((int)(s.amax[col] >> 23) - 127, -100) - 14;
        const float down = pow2_f32(-e / 2), rest = pow2_f32(-e - (-e / 2));
        if (sub == 0 && lane == 0) s.scale[col] = e;
        const uint32_t dst = smem + (uint32_t)((PAIR ? 2 * col : col) * layer_column_pitch(p.k));
        for (int c0 = sub * 32; c0 < chunks; c0 += each * 32) {
            const int c = c0 + lane;
            const bool ok = c < chunks;
            float v[8];
            layer_load8(base, dtype, vec, row + c * 8, ok, v);
            if (p.act_quant) {                          // (four lanes hold a block of 32: chunks come in fours)
                int ex;
                uint32_t lo, hi;
                act_quant8(v, ex, lo, hi);
                const uint32_t w[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
                const float up = pow2_f32(ex);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = f16_lo(w[i]) * up;
                    v[2 * i + 1] = f16_hi(w[i]) * up;
                }
            }
            if (!ok) continue;
            uint32_t a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = v[2 * i] * down * rest, x1 = v[2 * i + 1] * down * rest;
                a[i] = f16x2(x0, x1);
                if constexpr (PAIR) {
                    const float r0 = x0 - f16_lo(a[i]), r1 = x1 - f16_hi(a[i]);
                    b[i] = f16x2(fabsf(x0) < 65536.0f ? r0 : 0.0f, fabsf(x1) < 65536.0f ? r1 : 0.0f);   // (an infinity has no remainder)
                }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + c * 16), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]) : "memory");
            if constexpr (PAIR)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + c * 16 + layer_column_pitch(p.k)), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3]) : "memory");
        }
    }
    __syncthreads();
}

// Where a warp's copies are: the next chunk of K of a unit.
struct LayerSource {
    const uint8_t *wa, *wb, *sa, *sb;               // the unit's rows
    int unit, chunk;
};

// NT tiles of 8 columns, D stages a warp; FULL: K is whole chunks.
template <bool FIRST, bool PAIR, bool FULL, int NT, int D>
__global__ void __launch_bounds__(kLayerThreads, 1) layer_kernel(const __grid_constant__ LayerParams p) {
    extern __shared__ __align__(128) uint8_t layer_smem[];
    __shared__ LayerPlan s;
    const int tid = threadIdx.x, lane = tid & 31, warp = warp_id(), g = lane >> 2, tq = lane & 3;
    const uint32_t ring = smem_u32(layer_smem) + warp * D * kLayerStage, cols = smem_u32(layer_smem) + kLayerWarps * D * kLayerStage;
    const int column = layer_column_pitch(p.k);
    if constexpr (FIRST) {
        wait_predecessor();
        // The second kernel may begin: it reads the routes and the weights, which this wait has seen complete, before it
        // waits for this one.
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        for (int64_t i = (int64_t)blockIdx.x * kLayerThreads + tid; i < (int64_t)p.n * p.m; i += (int64_t)gridDim.x * kLayerThreads) p.count[i] = 0u;
    }
    layer_plan(s, p);
    const int chunks = (p.k + kLayerChunk - 1) / kLayerChunk, group = s.group, slice = warp % group, step = kLayerWarps / group;
    const int64_t kw = p.k / 2, ks = p.k / 32;
    LayerSource src{nullptr, nullptr, nullptr, nullptr, s.unit0 + warp / group, slice};
    auto seek = [&]() {                             // the rows of src.unit
        const int q = src.unit / p.units, u = src.unit - q * p.units;
        const int64_t e = s.expert[q];
        const int64_t ra = FIRST ? u * 8 : u * 16, rb = FIRST ? u * 8 : u * 16 + 8;
        src.wa = p.wa + e * p.wa_e + ra * kw;
        src.wb = p.wb + e * p.wb_e + rb * kw;
        src.sa = p.sa + e * p.sa_e + ra * ks;
        src.sb = p.sb + e * p.sb_e + rb * ks;
    };
    if (slice >= chunks) src.unit = s.unit1;        // (a short K has no share for this warp)
    if (src.unit < s.unit1) seek();
    // Copies the next chunk to a stage; a warp without one commits an empty group, so that groups count stages.
    auto request = [&](int stage) {
        if (src.unit < s.unit1) {
            const uint32_t to = ring + stage * kLayerStage;
            const int k0 = src.chunk * kLayerChunk;
            const int row = lane >> 3, part = lane & 7;
            if (FULL || k0 + part * 32 < p.k) {
                const int64_t off = row * kw + k0 / 2 + part * 16;
                const uint32_t at = to + row * kLayerPitch + part * 16;
                layer_copy16(at, src.wa + off);
                layer_copy16(at + 4 * kLayerPitch, src.wa + off + 4 * kw);
                layer_copy16(at + 8 * kLayerPitch, src.wb + off);
                layer_copy16(at + 12 * kLayerPitch, src.wb + off + 4 * kw);
            }
            // scales: the words that a row's 8 bytes lie in
            const uint32_t sto = to + 16 * kLayerPitch;
            if constexpr (FULL) {
                const int r = lane >> 1, w = lane & 1;
                layer_copy4(sto + r * 12 + w * 4, (r < 8 ? src.sa + r * ks : src.sb + (r - 8) * ks) + k0 / 32 + w * 4);
            } else {
                const int bytes = min(8, (p.k - k0) / 32);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int id = i * 32 + lane, r = id / 3, w = id - r * 3;
                    if (id < 48) {
                        const uintptr_t b = reinterpret_cast<uintptr_t>((r < 8 ? src.sa + r * ks : src.sb + (r - 8) * ks) + k0 / 32);
                        if ((int)(b & 3) + bytes > w * 4) layer_copy4(sto + r * 12 + w * 4, reinterpret_cast<const void *>((b & ~(uintptr_t)3) + w * 4));
                    }
                }
            }
            src.chunk += group;
            if (src.chunk >= chunks) {
                src.chunk = slice;
                src.unit += step;
                if (src.unit < s.unit1) seek();
            }
        }
        layer_commit();
    };
#pragma unroll
    for (int i = 0; i < D - 1; ++i) request(i);
    if constexpr (!FIRST) {
        wait_predecessor();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        // tokens without a route here
        for (int t = 0; t < p.m; ++t)
            if (!s.here[t])
                for (int i = blockIdx.x * kLayerThreads + tid; i < p.n; i += gridDim.x * kLayerThreads) store1(p.out, p.out_dtype, t * p.ldo + i, 0.0f);
    }
    int unit = s.unit0 + warp / group, stage = 0;
    for (int q = 0; q < s.passes; ++q) {
        layer_columns<PAIR>(s, p, q, FIRST, cols);
        const int n = s.routes[q], used = PAIR ? 2 * n : n, end = min(s.unit1, (q + 1) * p.units);
        for (; unit < end; unit += step) {
            float sum[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[j][i] = 0.0f;
            for (int chunk = slice; chunk < chunks; chunk += group) {
                layer_wait<D - 2>();
                __syncwarp();                       // all of this stage has come, and the one before it is free
                request(stage == 0 ? D - 1 : stage - 1);
                const uint32_t at = ring + stage * kLayerStage, sc = at + 16 * kLayerPitch;
                // scales of rows g and g + 8 (W1's and W3's row g): 8 bytes each
                uint32_t sa[2], sb[2];
                if constexpr (FULL) {
                    sa[0] = lds_u32(sc + g * 12); sa[1] = lds_u32(sc + g * 12 + 4);
                    sb[0] = lds_u32(sc + (g + 8) * 12); sb[1] = lds_u32(sc + (g + 8) * 12 + 4);
                } else {
                    const int u = unit - q * p.units;
                    const int64_t e = s.expert[q], ra = FIRST ? u * 8 : u * 16, rb = FIRST ? u * 8 : u * 16 + 8;
                    const int oa = (int)(reinterpret_cast<uintptr_t>(p.sa + e * p.sa_e + (ra + g) * ks + chunk * 8) & 3) * 8;
                    const int ob = (int)(reinterpret_cast<uintptr_t>(p.sb + e * p.sb_e + (rb + g) * ks + chunk * 8) & 3) * 8;
                    uint32_t a[3], b[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        a[i] = lds_u32(sc + g * 12 + i * 4);
                        b[i] = lds_u32(sc + (g + 8) * 12 + i * 4);
                    }
                    sa[0] = __funnelshift_r(a[0], a[1], oa); sa[1] = __funnelshift_r(a[1], a[2], oa);
                    sb[0] = __funnelshift_r(b[0], b[1], ob); sb[1] = __funnelshift_r(b[1], b[2], ob);
                }
                const int blocks = FULL ? 8 : min(8, (p.k - chunk * kLayerChunk) / 32);
                auto block = [&](int j, float s0, float s1) {
                    const uint32_t a = lds_u32(at + g * kLayerPitch + j * 16 + tq * 4), b = lds_u32(at + (g + 8) * kLayerPitch + j * 16 + tq * 4);
                    const uint32_t a0 = e2m1x2_byte_to_f16x2<0>(a), a1 = e2m1x2_byte_to_f16x2<1>(a), a2 = e2m1x2_byte_to_f16x2<2>(a), a3 = e2m1x2_byte_to_f16x2<3>(a);
                    const uint32_t b0 = e2m1x2_byte_to_f16x2<0>(b), b1 = e2m1x2_byte_to_f16x2<1>(b), b2 = e2m1x2_byte_to_f16x2<2>(b), b3 = e2m1x2_byte_to_f16x2<3>(b);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (t && used <= 8) break;
                        uint4 x = make_uint4(0u, 0u, 0u, 0u);
                        if (t * 8 + g < used) x = lds_u128(cols + (uint32_t)((t * 8 + g) * column + (chunk * kLayerChunk + j * 32 + tq * 8) * 2));
                        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        layer_mma(d, a0, b0, a1, b1, x.x, x.y);
                        layer_mma(d, a2, b2, a3, b3, x.z, x.w);
                        sum[t][0] = fmaf(d[0], s0, sum[t][0]);
                        sum[t][1] = fmaf(d[1], s0, sum[t][1]);
                        sum[t][2] = fmaf(d[2], s1, sum[t][2]);
                        sum[t][3] = fmaf(d[3], s1, sum[t][3]);
                    }
                };
                if (FULL || blocks == 8) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        block(j * 4, layer_scale<0>(sa[j]), layer_scale<0>(sb[j]));
                        block(j * 4 + 1, layer_scale<1>(sa[j]), layer_scale<1>(sb[j]));
                        block(j * 4 + 2, layer_scale<2>(sa[j]), layer_scale<2>(sb[j]));
                        block(j * 4 + 3, layer_scale<3>(sa[j]), layer_scale<3>(sb[j]));
                    }
                } else {
                    for (int j = 0; j < blocks; ++j) {
                        const uint32_t wa = (j < 4 ? sa[0] : sa[1]) >> (j & 3) * 8, wb = (j < 4 ? sb[0] : sb[1]) >> (j & 3) * 8;
                        block(j, layer_scale<0>(wa), layer_scale<0>(wb));
                    }
                }
                stage = stage == D - 1 ? 0 : stage + 1;
            }
            if (group > 1) {                        // shares of K: in the order of the warps
                const int bar = 1 + warp / group;
                if (slice)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s.red[warp][j * 4 + i][lane] = sum[j][i];
                asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(group * 32) : "memory");
                if (!slice)
                    for (int w = 1; w < group; ++w)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sum[j][i] += s.red[warp + w][j * 4 + i][lane];
                asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(group * 32) : "memory");
                if (slice) continue;
            }
            const int u = unit - q * p.units;
            if constexpr (FIRST) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int i = 0; i < (PAIR ? 1 : 2); ++i) {
                        const int r = PAIR ? j * 4 + tq : j * 8 + tq * 2 + i;
                        if (r >= n) continue;
                        const int e = s.scale[r], route = s.route[q][r];
                        const float lo = pow2_f32(e / 2), hi = pow2_f32(e - e / 2);
                        float gate = (PAIR ? sum[j][0] + sum[j][1] : sum[j][i]) * lo * hi, up = (PAIR ? sum[j][2] + sum[j][3] : sum[j][2 + i]) * lo * hi;
                        if (p.has_limit) {
                            gate = gate > p.limit ? p.limit : gate;                     // (a NaN stays one)
                            up = up > p.limit ? p.limit : up < -p.limit ? -p.limit : up;
                        }
                        p.h[(int64_t)route * (p.units * 8) + u * 8 + g] = p.weights[route] * (gate / (1.0f + expf(-gate)) * up);
                    }
                }
            } else {
                // a route's 16 results, then its arrival at the token's tile
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int r = j * 4 + tq;
                    if (r < n) {
                        const int e = s.scale[r];
                        const float lo = pow2_f32(e / 2), hi = pow2_f32(e - e / 2);
                        float *const to = p.part + (int64_t)s.route[q][r] * p.n + u * 16 + g;
                        __stcg(to, (sum[j][0] + sum[j][1]) * lo * hi);
                        __stcg(to + 8, (sum[j][2] + sum[j][3]) * lo * hi);
                    }
                }
                __threadfence();
                __syncwarp();
                bool last = false;
                if (lane < n) {
                    const int t = s.route[q][lane] / p.top_k;
                    last = atomicAdd(&p.count[(int64_t)u * p.m + t], 1u) == (uint32_t)s.here[t] - 1u;
                }
                uint32_t todo = __ballot_sync(0xffffffffu, last);
                __threadfence();
                while (todo) {                      // two tokens at a time
                    const int ra = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const int rb = todo ? __ffs(todo) - 1 : -1;
                    todo &= todo - 1;
                    const int r = lane < 16 ? ra : rb;
                    if (r >= 0) {
                        const int t = s.route[q][r] / p.top_k;
                        const float *from = p.part + (int64_t)t * p.top_k * p.n + u * 16 + (lane & 15);
                        float v[kLayerMaxTopK];
#pragma unroll
                        for (int j = 0; j < kLayerMaxTopK; ++j) v[j] = j < p.top_k && s.ids[t * p.top_k + j] >= 0 ? __ldcg(from + (int64_t)j * p.n) : 0.0f;
                        float y = 0.0f;
#pragma unroll
                        for (int j = 0; j < kLayerMaxTopK; ++j) y += v[j];
                        store1(p.out, p.out_dtype, t * p.ldo + u * 16 + (lane & 15), y);
                    }
                }
            }
        }
    }
    layer_wait<0>();
}

}  // namespace ws
