// Norms of queries and keys, head by head, and the rotation of positions, one pass:
//
//   u = x * rsqrt(mean(x^2) + eps) * (o + w)            over the d values of a head
//   a' = s (a cos - b sin),  b' = s (a sin + b cos)     for the pairs (a, b) of u's rotated part, angle = position * inv_freq
//
// The angle is a product of 64 bits, reduced to a turn before its cosine is taken in 32, so that positions of millions
// have the same error as the first ones.  A token's cosines and sines are computed once a block and serve all its heads.
#pragma once

#include "ws_values.cuh"

namespace ws {

constexpr int kHeadsThreads = 256;

struct HeadsParams {
    const void *x[2];                               // queries, keys
    void *y[2];
    const void *w[2];                               // [d] or null: 1
    int64_t ldt[2], ldh[2], ldyt[2], ldyh[2];       // elements from token to token, head to head
    int32_t heads[2];
    const void *positions;
    const float *inv_freq;                          // [pairs]
    int32_t m, d, pairs, start, interleaved, norm, dtype, w_dtype, position_bytes, lanes, groups;
    float eps, weight_offset, scale;
};

__device__ __forceinline__ void heads_angles(const HeadsParams &p, int t, float *cos_s, float *sin_s) {
    if (!p.pairs) return;
    const double at = p.position_bytes == 8 ? (double)static_cast<const int64_t *>(p.positions)[t] : (double)static_cast<const int32_t *>(p.positions)[t];
    for (int i = threadIdx.x; i < p.pairs; i += blockDim.x) {
        double turns = at * (double)p.inv_freq[i] * 0.15915494309189533577;     // 1 / (2 pi)
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        cos_s[i] = c * p.scale;
        sin_s[i] = s * p.scale;
    }
}

// Whole vectors of eight values.  A lane holds NU units of two vectors, those that are rotated into each other where
// halves are paired, so that a pair never leaves its lane; `lanes` neighbours hold a head.
template <bool F32, int NU>
__global__ void __launch_bounds__(kHeadsThreads) heads_kernel(const __grid_constant__ HeadsParams p) {
    __shared__ __align__(16) float cos_s[WS_MAX_PAIRS], sin_s[WS_MAX_PAIRS];
    const int t = blockIdx.x / p.groups, lane = threadIdx.x & (p.lanes - 1), per = kHeadsThreads / p.lanes;
    const int all = p.heads[0] + p.heads[1], step = per * p.groups;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // a unit's vectors (first values), -1: none; whether it is rotated
    int at[NU][2];
    bool turn[NU][2];
    const int rot = 2 * p.pairs, halves = p.interleaved ? 0 : p.pairs / 8;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = n * p.lanes + lane;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int v;
            if (u < halves) {
                v = p.start + u * 8 + h * p.pairs;
                turn[n][h] = true;
            } else {
                v = ((u - halves) * 2 + h) * 8;
                if (halves && v >= p.start) v += rot;
                turn[n][h] = p.interleaved && v >= p.start && v < p.start + rot;
            }
            at[n][h] = v < p.d ? v : -1;
        }
    }
    wait_predecessor();
    heads_angles(p, t, cos_s, sin_s);
    __syncthreads();
    for (int head = blockIdx.x % p.groups * per + threadIdx.x / p.lanes; head - (int)(threadIdx.x & 31) / p.lanes < all; head += step) {
        const bool ok = head < all;
        const int which = head >= p.heads[0], j = which ? head - p.heads[0] : head;
        const int64_t from = (int64_t)t * p.ldt[which] + (int64_t)j * p.ldh[which], to = (int64_t)t * p.ldyt[which] + (int64_t)j * p.ldyh[which];
        Eight<F32> raw[NU][2];
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) raw[n][h].load(p.x[which], from + (at[n][h] < 0 ? 0 : at[n][h]), ok && at[n][h] >= 0);
        float r = 1.0f;
        if (p.norm) {
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < NU; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = fmaf(raw[n][h].get(e), raw[n][h].get(e), sum);
            for (int o = p.lanes >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            r = rsqrtf(sum / (float)p.d + p.eps);
        }
        if (!ok) continue;
        const void *const w = p.w[which];
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            float v[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (w && at[n][h] >= 0) {
                    if (p.w_dtype == WS_ACT_F32) {
                        Eight<true> g;
                        g.load(w, at[n][h], true);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[h][e] = raw[n][h].get(e) * r * (p.weight_offset + g.get(e));
                    } else {
                        Eight<false> g;
                        g.load(w, at[n][h], true);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[h][e] = raw[n][h].get(e) * r * (p.weight_offset + g.get(e));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[h][e] = raw[n][h].get(e) * r;
                }
            }
            if (!p.interleaved && turn[n][0]) {
                const int i = at[n][0] - p.start;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float c = cos_s[i + e], s = sin_s[i + e], a = v[0][e], b = v[1][e];
                    v[0][e] = a * c - b * s;
                    v[1][e] = a * s + b * c;
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (at[n][h] < 0) continue;
                if (p.interleaved && turn[n][h]) {
                    const int i = (at[n][h] - p.start) / 2;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float c = cos_s[i + e / 2], s = sin_s[i + e / 2], a = v[h][e], b = v[h][e + 1];
                        v[h][e] = a * c - b * s;
                        v[h][e + 1] = a * s + b * c;
                    }
                }
                put8(p.y[which], F32 ? WS_ACT_F32 : WS_ACT_BF16, to + at[n][h], v[h]);
            }
        }
    }
}

// Any width, alignment and stride: a warp a head, read twice; a pair is one lane's.
__global__ void __launch_bounds__(kHeadsThreads) heads_any_kernel(const __grid_constant__ HeadsParams p) {
    __shared__ float cos_s[WS_MAX_PAIRS], sin_s[WS_MAX_PAIRS];
    const int t = blockIdx.x / p.groups, lane = threadIdx.x & 31, per = kHeadsThreads / 32, all = p.heads[0] + p.heads[1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    heads_angles(p, t, cos_s, sin_s);
    __syncthreads();
    const int rot = 2 * p.pairs;
    for (int head = blockIdx.x % p.groups * per + (threadIdx.x >> 5); head < all; head += per * p.groups) {
        const int which = head >= p.heads[0], j = which ? head - p.heads[0] : head;
        const int64_t from = (int64_t)t * p.ldt[which] + (int64_t)j * p.ldh[which], to = (int64_t)t * p.ldyt[which] + (int64_t)j * p.ldyh[which];
        float r = 1.0f;
        if (p.norm) {
            float sum = 0.0f;
            for (int i = lane; i < p.d; i += 32) {
                const float v = load1(p.x[which], p.dtype, from + i);
                sum = fmaf(v, v, sum);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            r = rsqrtf(sum / (float)p.d + p.eps);
        }
        auto value = [&](int i) {
            const float v = load1(p.x[which], p.dtype, from + i) * r;
            return p.w[which] ? v * (p.weight_offset + load1(p.w[which], p.w_dtype, i)) : v;
        };
        for (int i = lane; i < p.pairs; i += 32) {
            const int ia = p.start + (p.interleaved ? 2 * i : i), ib = ia + (p.interleaved ? 1 : p.pairs);
            const float a = value(ia), b = value(ib), c = cos_s[i], s = sin_s[i];
            store1(p.y[which], p.dtype, to + ia, a * c - b * s);
            store1(p.y[which], p.dtype, to + ib, a * s + b * c);
        }
        for (int i = lane; i < p.d - rot; i += 32) {
            const int v = i < p.start ? i : i + rot;
            store1(p.y[which], p.dtype, to + v, value(v));
        }
    }
}

}  // namespace ws
