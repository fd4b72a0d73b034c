// Norms of queries and keys, head by head, and the rotation of positions, one pass:
//
//   u = x * rsqrt(mean(x^2) + eps) * (o + w)            over the d values of a head
//   a' = s (a cos - b sin),  b' = s (a sin + b cos)     for the pairs (a, b) of u's rotated part, angle = position * inv_freq
//
// The angle is the whole product of position and frequency, in two numbers of 64 bits, reduced to a turn before its cosine is
// taken in 32, so that positions up to 2^53 have the same error as the first ones.  A token's cosines and sines are computed once a team of threads and serve all
// its heads: a lane keeps them, times the weights, for the pairs that it has of every head.
//
// Bound: HBM for many tokens (8192 tokens of 64 and 8 heads of 128 bf16 values 63 us, 4.8 TB/s; 12 instructions a value before
// a lane kept its factors, 8 now, are half of the issue slots), the launch for few (one token 5.3 us a call).  Widths,
// starts and strides that are no multiples of eight values are read value by value, twice.
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
    int32_t m, d, pairs, start, interleaved, norm, dtype, w_dtype, position_bytes;
    int32_t lanes, groups, teams;                   // lanes a head; blocks a token, or tokens a block
    float eps, weight_offset, scale;
};

__device__ __forceinline__ void heads_angles(const HeadsParams &p, int t, int tid, int threads, float *cos_s, float *sin_s) {
    if (!p.pairs || t >= p.m) return;
    const double at = p.position_bytes == 8 ? (double)static_cast<const int64_t *>(p.positions)[t] : (double)static_cast<const int32_t *>(p.positions)[t];
    for (int i = tid; i < p.pairs; i += threads) {
        // at * f = whole + rest exactly, and 1 / (2 pi) in two numbers: what is lost is below 2^-52 of a turn.
        constexpr double kTurn = 0.15915494309189535, kTurnRest = -9.839338337591243e-18;
        const double f = (double)p.inv_freq[i], whole = at * f, rest = fma(at, f, -whole);
        double turns = fma(whole, kTurn, -rint(whole * kTurn)) + fma(whole, kTurnRest, rest * kTurn);
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        cos_s[i] = c * p.scale;
        sin_s[i] = s * p.scale;
    }
}

// Whole vectors of eight values.  A lane holds NU units of two vectors, those that are rotated into each other where
// halves are paired, so that a pair never leaves its lane; `lanes` neighbours hold a head.  A team of threads has a token,
// or one of `groups` shares of its heads.
// WHOLE: every lane has all of its vectors.
template <bool F32, bool INTER, int NU, bool WHOLE>
__global__ void __launch_bounds__(kHeadsThreads, NU == 1 ? F32 ? 2 : 3 : 1) heads_kernel(const __grid_constant__ HeadsParams p) {
    __shared__ __align__(16) float cos_s[WS_MAX_PAIRS], sin_s[WS_MAX_PAIRS];      // of all teams: pairs * teams are no more
    const int threads = kHeadsThreads / p.teams, team = threadIdx.x / threads, tid = threadIdx.x - team * threads;
    const int t = p.teams > 1 ? blockIdx.x * p.teams + team : blockIdx.x / p.groups, share = p.teams > 1 ? 0 : blockIdx.x % p.groups;
    const int lane = tid & (p.lanes - 1), per = threads / p.lanes;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // a unit's vectors (first values), -1: none; whether it is rotated
    int at[NU][2];
    bool turn[NU][2];
    const int rot = 2 * p.pairs, halves = INTER ? 0 : p.pairs / 8;
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
                turn[n][h] = INTER && v >= p.start && v < p.start + rot;
            }
            at[n][h] = v < p.d ? v : -1;
        }
    }
    wait_predecessor();
    heads_angles(p, t, tid, threads, cos_s + team * p.pairs, sin_s + team * p.pairs);
    __syncthreads();
    const float over_d = 1.0f / (float)p.d;
    if (t >= p.m) return;                           // (whole warps: a team has 64 threads at least)
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const int heads = p.heads[which], mine = share * per + tid / p.lanes, first = share * per + (tid & ~31) / p.lanes;    // this lane's head, its warp's first
        if (first >= heads) continue;
        constexpr int kBytes = F32 ? 4 : 2;
        const int step = per * p.groups;
        const int64_t ahead = step * p.ldh[which] * kBytes, ahead_out = step * p.ldyh[which] * kBytes;
        const char *from = static_cast<const char *>(p.x[which]) + (t * p.ldt[which] + mine * p.ldh[which]) * kBytes;
        char *to = static_cast<char *>(p.y[which]) + (t * p.ldyt[which] + mine * p.ldyh[which]) * kBytes;
        Eight<F32> raw[NU][2];
        auto load = [&](bool there) {               // of the head at `from`
#pragma unroll
            for (int n = 0; n < NU; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (WHOLE) {
                        if (there) raw[n][h].load_all(from, at[n][h]);
                    } else {
                        raw[n][h].load(from, at[n][h] < 0 ? 0 : at[n][h], there && at[n][h] >= 0);
                    }
                }
        };
        load(mine < heads);
        // pairs (a, b) become (a fa - b fb, a fc + b fd); without rotation (a fa, b fd)
        float fa[NU][8], fb[NU][8], fc[NU][8], fd[NU][8];
#pragma unroll
        for (int n = 0; n < NU; ++n) {
            float w[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[h][e] = 1.0f;
                if (!p.w[which] || (!WHOLE && at[n][h] < 0)) continue;
                if (p.w_dtype == WS_ACT_F32) {
                    Eight<true> g;
                    g.load(p.w[which], at[n][h], true);
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[h][e] = p.weight_offset + g.get(e);
                } else {
                    Eight<false> g;
                    g.load(p.w[which], at[n][h], true);
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[h][e] = p.weight_offset + g.get(e);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float wa = INTER ? w[e / 4][e % 4 * 2] : w[0][e], wb = INTER ? w[e / 4][e % 4 * 2 + 1] : w[1][e];
                fa[n][e] = wa;
                fd[n][e] = wb;
                fb[n][e] = fc[n][e] = 0.0f;
                if (!turn[n][INTER ? e / 4 : 0]) continue;
                const int i = team * p.pairs + (INTER ? (at[n][e / 4] - p.start) / 2 + e % 4 : at[n][0] - p.start + e);
                const float c = cos_s[i], s = sin_s[i];
                fa[n][e] = wa * c;
                fb[n][e] = wb * s;
                fc[n][e] = wa * s;
                fd[n][e] = wb * c;
            }
        }
#pragma unroll 1
        for (int head = mine, lead = first; lead < heads; head += step, lead += step, to += ahead_out) {
            float v[NU][2][8];
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < NU; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[n][h][e] = raw[n][h].get(e);
                        sum = fmaf(v[n][h][e], v[n][h][e], sum);
                    }
            from += ahead;
            load(head + step < heads);              // the next head's, before this one's sum
            float r = 1.0f;
            if (p.norm) {
                for (int o = p.lanes >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                r = rsqrtf(sum * over_d + p.eps);
            }
            if (head >= heads) continue;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float &a = v[n][INTER ? e / 4 : 0][INTER ? e % 4 * 2 : e], &b = v[n][INTER ? e / 4 : 1][INTER ? e % 4 * 2 + 1 : e];
                    const float x = a * r, y = b * r;
                    a = x * fa[n][e];
                    b = y * fd[n][e];
                    if (turn[n][INTER ? e / 4 : 0]) {
                        a = fmaf(-y, fb[n][e], a);
                        b = fmaf(x, fc[n][e], b);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (WHOLE || at[n][h] >= 0) put8(to, F32 ? WS_ACT_F32 : WS_ACT_BF16, at[n][h], v[n][h]);
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
    heads_angles(p, t, threadIdx.x, kHeadsThreads, cos_s, sin_s);
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
