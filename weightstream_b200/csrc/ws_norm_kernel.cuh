// Norms before and after a block, with its gate, residual scale and the residual stream, one launch.
//
//   u = y                                       or  y * rsqrt(mean(y^2) + eps) * (o + w_post)
//   h = residual_scale * residual + block_scale * act(gate) * u
//   z = h * rsqrt(mean(h^2) + eps) * (o + w_next)
//
// All of it is held in 32 bits between the loads and the one rounding of h and of z to their types; z is taken from the
// unrounded h.
//
// Bound: HBM for many rows (8192 rows of 7168 with a gate a value: 131 us, 5.4 TB/s, in a graph of such calls 124 us; a
// row's two sums are the time in which its block loads nothing, so that several blocks share an SM), the launch for few
// (one row 2.7 us on the device).  Widths that no vector divides load value by value and are bound by those instructions
// (1503 rows of 2307: 10.3 us, 3.4 TB/s), and so are those beyond 16384, which besides read three times (2048 rows of 18432
// 256 us, of which HBM would need 58).
#pragma once

#include <type_traits>

#include "ws_device.cuh"

namespace ws {

struct NormParams {
    const void *y, *residual, *gate, *post_weight, *next_weight;
    void *hidden, *normed;
    int64_t ldy, ldr, ldg, ldh, ldn;   // elements a row; ldg 0: one gate for all rows
    int32_t m, n;
    int32_t gate_inc;                  // 1: a gate a value, 0: a gate a row
    int32_t y_dtype, r_dtype, g_dtype, w_dtype, h_dtype, n_dtype, gate_act;
    float weight_offset, eps, residual_scale, block_scale;
};

__device__ __forceinline__ float load1(const void *p, int dtype, int64_t i) {
    if (dtype == WS_ACT_F32) return static_cast<const float *>(p)[i];
    return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
}
__device__ __forceinline__ uint32_t bf16_bits(float v) {  // to nearest even
    uint16_t b;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(b) : "f"(v));
    return b;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {  // to nearest even, a in the low half
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ void store1(void *p, int dtype, int64_t i, float v) {
    if (dtype == WS_ACT_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)bf16_bits(v);
}
__device__ __forceinline__ float gate_value(float g, int act) { return act == WS_GATE_SIGMOID ? __fdividef(1.0f, 1.0f + __expf(-g)) : g; }

// The block's sum of v, the same on all threads.  `slot`: 32 floats of shared memory that the previous sum did not use.
__device__ __forceinline__ float block_sum(float v, float *slot) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? slot[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Eight values of a row as they are stored.  The loads are predicated instead of branched over: behind branches the
// compiler waits for one load before it issues the next (a row of 2307 values 15.8 us so, 1503 rows).
template <bool F32>
struct Eight {
    uint32_t w[F32 ? 8 : 4];  // consecutive values; fp32 rows are 32-byte aligned, bf16 rows 16
    __device__ __forceinline__ void load(const void *p, int64_t i, bool ok) {
#pragma unroll
        for (int e = 0; e < (F32 ? 8 : 4); ++e) w[e] = 0u;
        if constexpr (F32)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %9, 0;\n\t@p ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t}"
                         : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]), "+r"(w[4]), "+r"(w[5]), "+r"(w[6]), "+r"(w[7])
                         : "l"(static_cast<const float *>(p) + i), "r"((int)ok) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                         : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]) : "l"(static_cast<const uint16_t *>(p) + i), "r"((int)ok) : "memory");
    }
    __device__ __forceinline__ float get(int e) const {
        return __uint_as_float(F32 ? w[F32 ? e : 0] : e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    }
};
template <bool F32>
struct EightApart {
    uint32_t w[8];            // values `step` apart
    __device__ __forceinline__ void load(const void *p, int64_t i, int step, int left) {  // those before `left` are there
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e] = 0u;
            const int ok = e * step < left;
            if constexpr (F32)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}"
                             : "+r"(w[e]) : "l"(static_cast<const float *>(p) + i + e * step), "r"(ok) : "memory");
            else
                asm volatile("{\n\t.reg .pred p;\n\t.reg .b16 h;\n\tmov.b16 h, 0;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.b16 h, [%1];\n\tmov.b32 %0, {0, h};\n\t}"
                             : "=r"(w[e]) : "l"(static_cast<const uint16_t *>(p) + i + e * step), "r"(ok) : "memory");
        }
    }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(w[e]); }
};
__device__ __forceinline__ void put8(void *p, int dtype, int64_t i, const float (&v)[8]) {
    if (dtype == WS_ACT_F32) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(static_cast<float *>(p) + i), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
    } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
}

// A block a row, the row in registers: NV times eight values a thread.  VEC: eight consecutive ones; else (odd widths,
// strides or addresses) a block apart, so that a warp's loads are consecutive all the same.  RK, GK: kinds of the
// residual and of the gate (0: none, or for the gate one a row; 1: bf16, 2: fp32).  Everything that comes from HBM is
// requested before the first sum.
template <int NV, bool VEC, bool YF32, int RK, int GK>
__global__ void __launch_bounds__(NV == 1 ? 1024 : 512) block_norm_rows_kernel(const __grid_constant__ NormParams p) {
    __shared__ float slots[64];
    const int T = blockDim.x, tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    auto at = [&](int j) { return VEC ? (j * T + tid) * 8 : j * 8 * T + tid; };
    auto load = [&](auto &v, const void *q, int64_t row0, int j) {
        if constexpr (VEC) v.load(q, row0 + at(j), at(j) < p.n);
        else v.load(q, row0 + at(j), T, p.n - at(j));
    };
    auto weight = [&](const void *q, int j, float (&v)[8]) {
        if constexpr (VEC) {
            if (p.w_dtype == WS_ACT_F32) {
                Eight<true> r;
                r.load(q, at(j), at(j) < p.n);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = p.weight_offset + r.get(e);
            } else {
                Eight<false> r;
                r.load(q, at(j), at(j) < p.n);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = p.weight_offset + r.get(e);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = at(j) + e * T < p.n ? p.weight_offset + load1(q, p.w_dtype, at(j) + e * T) : 0.0f;
        }
    };
    auto store = [&](void *q, int dtype, int64_t row0, int j, const float (&v)[8]) {
        const int i = at(j);
        if (VEC) {
            if (i < p.n) put8(q, dtype, row0 + i, v);
        } else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e * T < p.n) store1(q, dtype, row0 + i + e * T, v[e]);
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    std::conditional_t<VEC, Eight<YF32>, EightApart<YF32>> y[NV];
    std::conditional_t<VEC, Eight<RK == 2>, EightApart<RK == 2>> r[NV];
    std::conditional_t<VEC, Eight<GK == 2>, EightApart<GK == 2>> g[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) load(y[j], p.y, row * p.ldy, j);
    if constexpr (RK != 0)
#pragma unroll
        for (int j = 0; j < NV; ++j) load(r[j], p.residual, row * p.ldr, j);
    if constexpr (GK != 0)
#pragma unroll
        for (int j = 0; j < NV; ++j) load(g[j], p.gate, row * p.ldg, j);
    float f = p.block_scale;
    if (GK == 0 && p.gate) f *= gate_value(load1(p.gate, p.g_dtype, row * p.ldg), p.gate_act);
    const float inv_n = 1.0f / (float)p.n;
    float h[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) h[j][e] = y[j].get(e);
    if (p.post_weight) {
        float w[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j) weight(p.post_weight, j, w[j]);
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(h[j][e], h[j][e], s);
        f *= rsqrtf(fmaf(block_sum(s, slots), inv_n, p.eps));
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[j][e] *= w[j][e];
    }
    float w[NV][8];
    if (p.normed)
#pragma unroll
        for (int j = 0; j < NV; ++j) weight(p.next_weight, j, w[j]);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[j][e] *= f;
            if constexpr (GK != 0) h[j][e] *= gate_value(g[j].get(e), p.gate_act);
            if constexpr (RK != 0) h[j][e] = fmaf(p.residual_scale, r[j].get(e), h[j][e]);
            s = fmaf(h[j][e], h[j][e], s);
        }
        if (p.hidden) store(p.hidden, p.h_dtype, row * p.ldh, j, h[j]);
    }
    if (!p.normed) return;
    const float next = rsqrtf(fmaf(block_sum(s, slots + 32), inv_n, p.eps));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[j][e] *= next * w[j][e];
        store(p.normed, p.n_dtype, row * p.ldn, j, h[j]);
    }
}

// Any width, any alignment: a block a row, three passes over it (L2 serves the second and third).  The last pass reads
// each value and writes its results on one thread, so that the stream may be updated in place.
__global__ void __launch_bounds__(512) block_norm_any_kernel(const __grid_constant__ NormParams p) {
    __shared__ float slots[64];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    const int64_t row = blockIdx.x;
    const float inv_n = 1.0f / (float)p.n;
    float post = 1.0f;
    if (p.post_weight) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float v = load1(p.y, p.y_dtype, row * p.ldy + i);
            s = fmaf(v, v, s);
        }
        post = rsqrtf(fmaf(block_sum(s, slots), inv_n, p.eps));
    }
    auto value = [&](int i) {
        float u = load1(p.y, p.y_dtype, row * p.ldy + i);
        if (p.post_weight) u *= post * (p.weight_offset + load1(p.post_weight, p.w_dtype, i));
        u *= p.block_scale;
        if (p.gate) u *= gate_value(load1(p.gate, p.g_dtype, row * p.ldg + (int64_t)i * p.gate_inc), p.gate_act);
        return p.residual ? fmaf(p.residual_scale, load1(p.residual, p.r_dtype, row * p.ldr + i), u) : u;
    };
    float next = 0.0f;
    if (p.normed) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float h = value(i);
            s = fmaf(h, h, s);
        }
        next = rsqrtf(fmaf(block_sum(s, slots + 32), inv_n, p.eps));
    }
    for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
        const float h = value(i);
        if (p.hidden) store1(p.hidden, p.h_dtype, row * p.ldh + i, h);
        if (p.normed) store1(p.normed, p.n_dtype, row * p.ldn + i, h * next * (p.weight_offset + load1(p.next_weight, p.w_dtype, i)));
    }
}

}  // namespace ws
