// Low-rank adapters of many requests beside a shared projection:  out[t] = y[t] + scale[id] * B[id] (A[id] x[t]).
//
// Up to 512 tokens, a tile is up to 8 * NT tokens of one adapter.  A cluster of blocks takes a tile: every block shrinks
// a slice of K (S = A x^T, ranks as the rows of the product and tokens as its columns), stores its sums into all blocks'
// shared memory, and expands the whole S to a slice of N (B S).  So a call is one launch without workspace or atomics on
// results; the sums' order depends on the sizes alone.  More tokens are sorted by adapter and run as two products
// (below).
//
// Both products are bf16 mma.sync with fp32 accumulators.  In the cluster's form they are fed straight from global
// memory: the order of a contraction's terms is free, so a lane takes 8 consecutive values of a row, 16 bytes, as the
// terms that the instruction's fragment layout gives it (4 lanes x 16 bytes are two whole sectors of a row), and no
// shared memory or shuffles lie between.  mma.sync's rate is enough at the ranks in use: 2 m r (k + n) operations, three
// times that where an operand is split, against m (2 k + 8 n) bytes; 4000 rows of rank 64 keep it busy for 30 us and
// HBM for 47.
//
// Bound: latency for few tokens (one row of 8192 x 7168 at rank 16 5.7 us, 64 rows of 24 adapters 9.7 us, of which HBM
// needs 2.5: finding the tile, two waits for HBM and the blocks' meeting follow one another).  For prompts HBM would be
// (4000 rows of rank 64: 96 us, 3.2 TB/s; each by itself on cold caches, the plan takes 9, the first product 29 and the
// second 63).
//
// fp32 operands (x, and S between the products) are split into three bf16 parts that add up to all 24 bits, and each
// part is multiplied: nothing is rounded to 16 bits but the weights that are stored so.  An infinite activation has no
// second and third part.  A weight that is not finite makes its results NaN where a part is zero, also those that the
// definition makes infinite.
#pragma once

#include <cooperative_groups.h>

#include "ws_norm_kernel.cuh"

namespace ws {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraMaxCluster = 8;
// Up to this many tokens a block finds its tile by itself.  This form and the sorted one, K 8192, N 7168, us: rank 16, 256
// tokens of one request 14 and 20, 512 of one 18 and 24, of 24 adapters 27 and 27, of 200 54 and 83; 1024 tokens of one 39
// and 27, of 24 47 and 35.  At rank 64, 512 tokens of 200 adapters 157 and 196, but 256 of one 32 and 26, 512 of one 54 and
// 34: few adapters of high rank would be sorted earlier, which a limit on tokens alone does not do.
constexpr int kLoraDirect = 512;
constexpr int kLoraMaxAdapters = 16384;      // of a sorted batch: three words of shared memory each, of 227 KB

struct LoraTile {
    int32_t adapter, start, count, pad;      // adapter -1: tokens without one
};
struct LoraParams {
    const void *x, *y;
    void *out;
    const uint16_t *a, *b;
    const int32_t *ids;
    const float *scale;        // or null: 1
    const float *s_in;         // [m, r] shrunk rows to expand, or null: shrink x
    float *s_out;              // [m, r] where shrunk rows go instead of being expanded, or null
    int64_t ldx, ldy, ldo;
    int32_t m, k, n, r, adapters;
    int32_t y_dtype, cluster;
    // sorted batches
    int32_t *tiles_count, *perm;   // tiles_count: of all tiles, of those of an adapter
    LoraTile *tiles;
    int32_t tile, skip_none, most;   // most: the first product's largest cut, as a power of two
};

__device__ __forceinline__ int lora_id(const LoraParams &p, int t) {
    const int id = p.ids[t];
    return id >= 0 && id < p.adapters ? id : -1;
}

// More tokens than a block looks through: they are grouped by adapter first.  The order of tokens within a group is the
// atomics'; a token's result does not depend on its place in a tile.
__global__ void __launch_bounds__(1024) lora_plan_kernel(const __grid_constant__ LoraParams p) {
    extern __shared__ int32_t lora_hist[];
    int32_t *count = lora_hist, *first = lora_hist + p.adapters + 1;  // tokens of a bucket; its first place
    int32_t *tile0 = first + p.adapters + 1;                          // its first tile
    __shared__ int32_t warp_sum[32][2];
    const int tid = threadIdx.x, lane = tid & 31, buckets = p.adapters + 1;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int i = tid; i < buckets; i += 1024) count[i] = 0;
    wait_predecessor();
    __syncthreads();
    // (one atomic for all of a warp's tokens of an adapter: a prompt's tokens would queue for one word otherwise)
    constexpr int kBatch = 4;  // ids a thread requests together
    int id[kBatch];
    auto request = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) id[i] = t0 + i * 1024 + tid < p.m ? lora_id(p, t0 + i * 1024 + tid) : -2;
    };
    for (int t0 = 0; t0 < p.m; t0 += kBatch * 1024) {
        request(t0);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const uint32_t alike = __match_any_sync(0xffffffffu, id[i]);
            if (id[i] != -2 && (alike & ((1u << lane) - 1)) == 0) atomicAdd(&count[id[i] < 0 ? p.adapters : id[i]], __popc(alike));
        }
    }
    __syncthreads();
    const int per = (buckets + 1023) / 1024, b0 = tid * per, b1 = min(buckets, b0 + per);
    int32_t tok = 0, til = 0;
    for (int b = b0; b < b1; ++b) {
        tok += count[b];
        if (b < p.adapters || !p.skip_none) til += (count[b] + p.tile - 1) / p.tile;
    }
    int32_t st = tok, sl = til;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, st, o), v = __shfl_up_sync(0xffffffffu, sl, o);
        if (lane >= o) {
            st += u;
            sl += v;
        }
    }
    if (lane == 31) {
        warp_sum[tid >> 5][0] = st;
        warp_sum[tid >> 5][1] = sl;
    }
    __syncthreads();
    int32_t before_tok = st - tok, before_til = sl - til;
    for (int w = 0; w < (tid >> 5); ++w) {
        before_tok += warp_sum[w][0];
        before_til += warp_sum[w][1];
    }
    if (tid == 1023) *p.tiles_count = before_til + til;
    for (int b = b0; b < b1; ++b) {
        const int c = count[b];
        first[b] = before_tok;
        tile0[b] = before_til;
        if (b == p.adapters) p.tiles_count[1] = before_til;
        before_tok += c;
        if (b < p.adapters || !p.skip_none) before_til += (c + p.tile - 1) / p.tile;
    }
    __syncthreads();
    for (int t0 = 0; t0 < p.m; t0 += kBatch * 1024) {
        if (p.m > kBatch * 1024) request(t0);  // (else they are still there)
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int b = id[i] < 0 ? p.adapters : id[i];
            const uint32_t alike = __match_any_sync(0xffffffffu, id[i]);
            int left = 0;
            if (id[i] != -2 && (alike & ((1u << lane) - 1)) == 0) left = atomicSub(&count[b], __popc(alike));   // the bucket's size, less each time
            left = __shfl_sync(0xffffffffu, left, __ffs(alike) - 1) - __popc(alike & ((1u << lane) - 1));
            if (id[i] == -2 || (b == p.adapters && p.skip_none)) continue;
            const int c = (b + 1 < buckets ? first[b + 1] : p.m) - first[b], at = c - left;
            p.perm[first[b] + at] = t0 + i * 1024 + tid;
            if (at % p.tile == 0) p.tiles[tile0[b] + at / p.tile] = LoraTile{id[i], first[b] + at, min(p.tile, c - at), 0};
        }
    }
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The leading eight bits of two floats as bf16 (a in the low half); the floats keep the rest.  Cut off, not rounded, so that
// no finite value becomes infinite; an infinite one leaves nothing.
__device__ __forceinline__ float after_bf16(float v) { return fabsf(v) == __uint_as_float(0x7F800000u) ? 0.0f : v - __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t cut_bf16x2(float &a, float &b) {
    const uint32_t r = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    a = after_bf16(a);
    b = after_bf16(b);
    return r;
}

// Eight consecutive values of a bf16 row from `i`, those from `limit` on as zeros.  VEC: `limit` is a multiple of 8 and
// the row 16-byte aligned.
// (Predicated loads: behind branches the compiler waits for one before it issues the next.)
__device__ __forceinline__ uint4 load16_if(const void *p, bool ok) {
    uint4 r = make_uint4(0, 0, 0, 0);
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w) : "l"(p), "r"((int)ok));
    return r;
}
__device__ __forceinline__ uint2 load8_if(const void *p, bool ok) {
    uint2 r = make_uint2(0, 0);
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t@p ld.global.nc.v2.b32 {%0, %1}, [%2];\n\t}" : "+r"(r.x), "+r"(r.y) : "l"(p), "r"((int)ok));
    return r;
}
template <bool VEC>
__device__ __forceinline__ uint4 row8(const uint16_t *row, int i, int limit) {
    if (VEC) return load16_if(row + i, i < limit);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w[j] = (i + 2 * j < limit ? (uint32_t)__ldg(row + i + 2 * j) : 0u) | (i + 2 * j + 1 < limit ? (uint32_t)__ldg(row + i + 2 * j + 1) << 16 : 0u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool VEC>
__device__ __forceinline__ void row8(const float *row, int i, int limit, float (&v)[8]) {
    if (VEC) {
        const uint4 a = load16_if(row + i, i < limit), b = load16_if(row + i + 4, i < limit);
        v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i + j < limit ? __ldg(row + i + j) : 0.0f;
    }
}

// Four consecutive values of a token's y as they are stored, as numbers, and of its result.  tok < 0: none.
template <bool VEC>
__device__ __forceinline__ uint4 get4(const LoraParams &p, int64_t tok, int nn) {
    const bool f32 = p.y_dtype == WS_ACT_F32, ok = tok >= 0 && nn < p.n;
    const int64_t at = ok ? tok * p.ldy + nn : 0;
    uint4 r = make_uint4(0, 0, 0, 0);
    if (VEC) {
        // (y may be out: not a read-only load)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
                     "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t@q ld.global.v2.b32 {%0, %1}, [%4];\n\t}"
                     : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
                     : "l"(static_cast<const char *>(p.y) + at * (f32 ? 4 : 2)), "r"((int)(ok && f32)), "r"((int)(ok && !f32)) : "memory");
    } else if (ok) {
        uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (nn + j < p.n) v[j] = __float_as_uint(load1(p.y, p.y_dtype, at + j));
        r = make_uint4(v[0], v[1], v[2], v[3]);
    }
    return r;
}
template <bool VEC>
__device__ __forceinline__ void numbers4(const LoraParams &p, const uint4 &r, float (&v)[4]) {
    const bool bf16 = VEC && p.y_dtype != WS_ACT_F32;
    v[0] = __uint_as_float(bf16 ? r.x << 16 : r.x);
    v[1] = __uint_as_float(bf16 ? r.x & 0xFFFF0000u : r.y);
    v[2] = __uint_as_float(bf16 ? r.y << 16 : r.z);
    v[3] = __uint_as_float(bf16 ? r.y & 0xFFFF0000u : r.w);
}
template <bool VEC>
__device__ __forceinline__ void put4(const LoraParams &p, int64_t tok, int nn, const float (&v)[4]) {
    if (nn >= p.n) return;
    if (VEC && p.y_dtype == WS_ACT_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + tok * p.ldo + nn) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (VEC) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + tok * p.ldo + nn) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (nn + j < p.n) store1(p.out, p.y_dtype, tok * p.ldo + nn + j, v[j]);
    }
}

// Tokens without an adapter: their y as it is, or zeros for shrunk rows.  A block's slice of all of them, a warp a token.
template <bool VEC>
__device__ __forceinline__ void lora_none(const LoraParams &p, const int32_t *toks, int most, int part, int parts) {
    const int n = p.s_out ? p.r : VEC ? p.n / 4 : p.n, n0 = (int)((int64_t)n * part / parts), n1 = (int)((int64_t)n * (part + 1) / parts);
    if (!p.s_out && p.out == p.y && p.ldo == p.ldy) return;
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < most; i += kLoraWarps) {  // a warp a token
        const int64_t tok = toks[i];
        if (tok < 0) break;
        if (p.s_out) {
            for (int j = n0 + lane; j < n1; j += 32) p.s_out[tok * p.r + j] = 0.0f;
        } else if (VEC) {
            for (int j0 = n0 + lane; j0 < n1; j0 += 8 * 32) {
                uint4 v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = get4<true>(p, j0 + u * 32 < n1 ? tok : -1, (j0 + u * 32) * 4);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (j0 + u * 32 >= n1) break;
                    float f[4];
                    numbers4<VEC>(p, v[u], f);
                    put4<true>(p, tok, (j0 + u * 32) * 4, f);
                }
            }
        } else {
            for (int j = n0 + lane; j < n1; j += 32) store1(p.out, p.y_dtype, tok * p.ldo + j, load1(p.y, p.y_dtype, tok * p.ldy + j));
        }
    }
}

// The tokens of tile number `tile` and their adapter; false: there are fewer tiles.  A token leads a tile if the number of
// earlier tokens with its adapter is a multiple of the tile's size; tiles are numbered by their leaders' places, so the
// blocks that have work come first.
template <int TOKENS>
__device__ __forceinline__ bool find_tile(const LoraParams &p, int tile, uint8_t *scratch, int32_t *toks, int &adapter) {
    constexpr int H = kLoraDirect / kLoraThreads;   // tokens a thread looks after
    constexpr int kSlots = 2 * kLoraDirect, kChunks = kLoraDirect / 32;
    int32_t *const slots = reinterpret_cast<int32_t *>(scratch);                                           // a hash table of the ids that occur
    auto *const held = reinterpret_cast<uint8_t(*)[kSlots]>(scratch + kSlots * 4);                         // how many of 32 consecutive tokens have that id
    __shared__ uint32_t leads[kChunks];
    __shared__ int32_t lead_id, lead_before;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int id[H], before[H];
#pragma unroll
    for (int h = 0; h < H; ++h) id[h] = tid + h * kLoraThreads < p.m ? lora_id(p, tid + h * kLoraThreads) : -2;
    if (tid < TOKENS) toks[tid] = -1;
    if (p.m > 32) {
        for (int i = tid; i < kSlots / 4; i += kLoraThreads) reinterpret_cast<int4 *>(slots)[i] = make_int4(-3, -3, -3, -3);
        for (int i = tid; i < kChunks * kSlots / 16; i += kLoraThreads) reinterpret_cast<uint4 *>(held)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    int slot[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const uint32_t alike = __match_any_sync(0xffffffffu, id[h]);
        before[h] = __popc(alike & ((1u << lane) - 1));
        if (p.m > 32 && h * kLoraThreads < p.m) {
            slot[h] = (int)((uint32_t)id[h] * 2654435761u >> 16) % kSlots;
            for (;;) {  // ends: there are twice as many slots as tokens
                const int32_t o = atomicCAS(&slots[slot[h]], -3, id[h]);
                if (o == -3 || o == id[h]) break;
                slot[h] = (slot[h] + 1) % kSlots;
            }
            if ((alike & ((1u << lane) - 1)) == 0) held[h * kLoraWarps + warp][slot[h]] = (uint8_t)__popc(alike);
        }
    }
    if (p.m > 32) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < H; ++h)
            if (h * kLoraThreads < p.m)
                for (int c = 0; c < h * kLoraWarps + warp; ++c) before[h] += held[c][slot[h]];
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const bool leader = id[h] != -2 && before[h] % TOKENS == 0 && !(id[h] == -1 && p.skip_none);
        const uint32_t all = __ballot_sync(0xffffffffu, leader);
        if (lane == 0) leads[h * kLoraWarps + warp] = all;
    }
    __syncthreads();
    int count = 0;
    for (int w = 0; w < kLoraDirect / 32; ++w) {
        const uint32_t all = leads[w];
        const int n = __popc(all);
        if (tile >= count && tile < count + n && (w % kLoraWarps) == warp && (all >> lane & 1) && __popc(all & ((1u << lane) - 1)) == tile - count) {
            lead_id = id[w / kLoraWarps];
            lead_before = before[w / kLoraWarps];
        }
        count += n;
    }
    if (tile >= count) return false;
    __syncthreads();
    adapter = lead_id;
#pragma unroll
    for (int h = 0; h < H; ++h)
        if (id[h] == adapter && before[h] >= lead_before && before[h] < lead_before + TOKENS) toks[before[h] - lead_before] = tid + h * kLoraThreads;
    return true;
}

template <int RT, int NT>
struct LoraShape {
    static constexpr int kTokens = NT * 8, kRanks = RT * 16;
    static constexpr int kSums = RT * NT * 128;                              // values of S
    // a token's ranks in bf16, padded so that a warp's fragment loads meet no bank twice
    static constexpr int kRow = kRanks * 2 + (RT >= 4 ? 64 : 0);
    static constexpr int kSplit = 3 * kTokens * kRow;
    static constexpr int kFind = kLoraDirect * 8 + kLoraDirect / 32 * kLoraDirect * 2;    // find_tile's tables
    static constexpr int kWork = kLoraWarps * kSums * 4 > kSplit ? kLoraWarps * kSums * 4 : kSplit;
    static constexpr int kScratch = kWork > kFind ? kWork : kFind;
    static constexpr int kSmem = kScratch + kLoraMaxCluster * kSums * 4;
    static constexpr int kAhead = RT * NT <= 2 ? 4 : RT * NT <= 8 ? 2 : 1;   // steps of K requested together
};

template <int RT, int NT, bool XF32, bool VEC>
__global__ void __launch_bounds__(kLoraThreads, RT == 1 ? 2 : 1) lora_kernel(const __grid_constant__ LoraParams p) {
    namespace cg = cooperative_groups;
    using S = LoraShape<RT, NT>;
    extern __shared__ __align__(16) uint8_t lora_smem[];  // find_tile's tables, then the warps' sums, then the split S; the blocks' sums
    float *const warps = reinterpret_cast<float *>(lora_smem);                      // [warp][kSums], then the split S
    float *const sums = reinterpret_cast<float *>(lora_smem + S::kScratch);         // the S of the cluster's blocks, [block][kSums]
    __shared__ int32_t toks[S::kTokens];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int C = p.cluster, part = blockIdx.x % C, tile = blockIdx.x / C;
    cg::cluster_group cl = cg::this_cluster();
    const bool meets = C > 1 && !p.s_in;
    if (meets) cl.barrier_arrive();  // waited for before another block's shared memory is written
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();

    // ---- the tile's tokens
    int adapter;
    if (p.tiles) {
        if (tile >= *p.tiles_count) return;
        const LoraTile q = p.tiles[tile];
        adapter = q.adapter;
        if (tid < S::kTokens) toks[tid] = tid < q.count ? p.perm[q.start + tid] : -1;
    } else if (!find_tile<S::kTokens>(p, tile, lora_smem, toks, adapter)) {
        return;  // (the same on all threads of the cluster)
    }
    __syncthreads();
    if (adapter < 0) {  // nothing to add
        lora_none<VEC>(p, toks, S::kTokens, part, C);
        return;
    }

    // ---- S = A x^T over this block's K, a step of 32 a warp
    if (!p.s_in) {
        float acc[RT][NT][4] = {};
        const uint16_t *arow[RT][2];
        bool aok[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = i * 16 + h * 8 + g;
                aok[i][h] = row < p.r;
                arow[i][h] = p.a + ((int64_t)adapter * p.r + min(row, p.r - 1)) * p.k;
            }
        const char *xrow[NT];
        bool xok[NT];
#pragma unroll
        for (int q = 0; q < NT; ++q) {
            const int tok = toks[q * 8 + g];
            xok[q] = tok >= 0;
            xrow[q] = static_cast<const char *>(p.x) + (int64_t)max(tok, 0) * p.ldx * (XF32 ? 4 : 2);
        }
        const int steps = (p.k + 31) / 32, s0 = (int)((int64_t)steps * part / C), s1 = (int)((int64_t)steps * (part + 1) / C);
        constexpr int U = S::kAhead;
        for (int st = s0 + warp; st < s1; st += kLoraWarps * U) {
            uint4 aw[U][RT][2], xw[U][NT];
            float xf[XF32 ? U : 1][NT][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k0 = (st + u * kLoraWarps) * 32 + t4 * 8, limit = st + u * kLoraWarps < s1 ? p.k : 0;
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) aw[u][i][h] = row8<VEC>(arow[i][h], k0, aok[i][h] ? limit : 0);
#pragma unroll
                for (int q = 0; q < NT; ++q) {
                    if (XF32) row8<VEC>(reinterpret_cast<const float *>(xrow[q]), k0, xok[q] ? limit : 0, xf[u % (XF32 ? U : 1)][q]);
                    else xw[u][q] = row8<VEC>(reinterpret_cast<const uint16_t *>(xrow[q]), k0, xok[q] ? limit : 0);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int part3 = 0; part3 < (XF32 ? 3 : 1); ++part3)
#pragma unroll
                    for (int q = 0; q < NT; ++q) {
                        uint4 xv;
                        if (XF32) {
                            float(&f)[8] = xf[u % (XF32 ? U : 1)][q];
                            xv = make_uint4(cut_bf16x2(f[0], f[1]), cut_bf16x2(f[2], f[3]), cut_bf16x2(f[4], f[5]), cut_bf16x2(f[6], f[7]));
                        } else {
                            xv = xw[u][q];
                        }
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            const uint4 &lo = aw[u][i][0], &hi = aw[u][i][1];
                            mma_bf16(acc[i][q], lo.x, hi.x, lo.y, hi.y, xv.x, xv.y);
                            mma_bf16(acc[i][q], lo.z, hi.z, lo.w, hi.w, xv.z, xv.w);
                        }
                    }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int q = 0; q < NT; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) warps[warp * S::kSums + ((i * NT + q) * 4 + e) * 32 + lane] = acc[i][q][e];
        __syncthreads();
        if (meets) cl.barrier_wait();
        for (int j = tid; j < S::kSums; j += kLoraThreads) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kLoraWarps; ++w) s += warps[w * S::kSums + j];
            for (int c = 0; c < C; ++c) (meets ? cl.map_shared_rank(sums, c) : sums)[part * S::kSums + j] = s;
        }
    }

    // ---- this warp's first 64 rows of B and its tokens' y are on their way while the blocks meet
    constexpr int KP = RT >= 2 ? RT / 2 : 1;   // steps of 32 ranks (of 16 for RT = 1)
    const int blocks = (p.n + 63) / 64, nb1 = p.s_out ? 0 : (int)((int64_t)blocks * (part + 1) / C);
    int nb = (int)((int64_t)blocks * part / C) + warp;
    uint4 bw[4][2][KP];
    uint4 yv[NT][4];
    int mytok[NT][2];                          // the tokens of this lane's results
#pragma unroll
    for (int q = 0; q < NT; ++q) {
        mytok[q][0] = toks[q * 8 + t4 * 2];
        mytok[q][1] = toks[q * 8 + t4 * 2 + 1];
    }
    auto request = [&]() {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = nb * 64 + h * 32 + g * 4 + j;
                const uint16_t *b = p.b + ((int64_t)adapter * p.n + min(row, p.n - 1)) * p.r;
                const int limit = row < p.n ? p.r : 0;
                if (RT >= 2) {
#pragma unroll
                    for (int q = 0; q < KP; ++q) bw[j][h][q] = row8<VEC>(b, q * 32 + t4 * 8, limit);
                } else if (VEC) {
                    const uint2 v = load8_if(b + t4 * 4, t4 * 4 < limit);
                    bw[j][h][0] = make_uint4(v.x, v.y, 0, 0);
                } else {
                    bw[j][h][0] = row8<false>(b, t4 * 4, min(limit, t4 * 4 + 4));
                }
            }
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                yv[q][e] = get4<VEC>(p, mytok[q][e & 1], nb * 64 + (e >> 1) * 32 + g * 4);
            }
    };
    if (meets) cl.barrier_arrive();  // (before the loads: it would wait for them)
    if (nb < nb1) request();
    if (meets) cl.barrier_wait();
    else __syncthreads();

    // ---- the whole S: the cluster's slices in order, in three bf16 parts of scale * S
    uint8_t *const split = lora_smem;
    const float scale = p.scale && !p.s_out ? p.scale[adapter] : 1.0f;
    const int j0 = p.s_out ? S::kSums * part / C : 0, j1 = p.s_out ? S::kSums * (part + 1) / C : S::kSums;
    for (int j = j0 + tid; j < j1; j += kLoraThreads) {
        const int l = j & 31, e = (j >> 5) & 3, iq = j >> 7, i = iq / NT, q = iq % NT;
        const int rank = i * 16 + (l >> 2) + (e >> 1) * 8, place = q * 8 + (l & 3) * 2 + (e & 1), tok = toks[place];
        float s = 0.0f;
        if (p.s_in) {
            if (tok >= 0 && rank < p.r) s = p.s_in[(int64_t)tok * p.r + rank];
        } else {
            for (int c = 0; c < C; ++c) s += sums[c * S::kSums + j];
        }
        if (p.s_out) {
            if (tok >= 0 && rank < p.r) p.s_out[(int64_t)tok * p.r + rank] = s;
            continue;
        }
        s = rank < p.r ? s * scale : 0.0f;  // (A's missing rows are zeros, which an infinite activation makes NaN)
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            *reinterpret_cast<uint16_t *>(split + (w * S::kTokens + place) * S::kRow + rank * 2) = (uint16_t)(__float_as_uint(s) >> 16);
            s = after_bf16(s);
        }
    }
    __syncthreads();

    // ---- out = y + B S over this block's N, 64 rows of B a warp: row h * 32 + g * 4 + j of them is row h * 8 + g of
    // product j, so that a lane ends with four consecutive outputs
    while (nb < nb1) {
        float acc[NT][4][4] = {};
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                const uint8_t *srow = split + (w * S::kTokens + q * 8 + g) * S::kRow;
#pragma unroll
                for (int kp = 0; kp < KP; ++kp) {
                    if (RT >= 2) {
                        const uint4 s = *reinterpret_cast<const uint4 *>(srow + kp * 64 + t4 * 16);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            mma_bf16(acc[q][j], bw[j][0][kp].x, bw[j][1][kp].x, bw[j][0][kp].y, bw[j][1][kp].y, s.x, s.y);
                            mma_bf16(acc[q][j], bw[j][0][kp].z, bw[j][1][kp].z, bw[j][0][kp].w, bw[j][1][kp].w, s.z, s.w);
                        }
                    } else {
                        const uint2 s = *reinterpret_cast<const uint2 *>(srow + t4 * 8);
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma_bf16(acc[q][j], bw[j][0][0].x, bw[j][1][0].x, bw[j][0][0].y, bw[j][1][0].y, s.x, s.y);
                    }
                }
            }
        float sum[NT][4][4];
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                numbers4<VEC>(p, yv[q][e], sum[q][e]);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[q][e][j] += acc[q][j][e];
            }
        const int at = nb * 64 + g * 4;
        nb += kLoraWarps;
        if (nb < nb1) request();
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (mytok[q][e & 1] >= 0) put4<VEC>(p, mytok[q][e & 1], at + (e >> 1) * 32, sum[q][e]);
            }
    }
}

// ---------------------------------------------------------------- sorted batches
// Prompts: tiles of 64 tokens of one adapter, the two products as two launches, each a stream over its large operand
// (x; y and out), with the shrunk rows between them in the workspace.
constexpr int kSortTokens = 64;
constexpr int kSortK = 128;                   // values of K a stage holds

template <int RT, bool XF32>
struct ShrinkShape {
    static constexpr int kX = kSortTokens * kSortK * (XF32 ? 4 : 2), kStage = kX + RT * 16 * kSortK * 2;
    static constexpr int kStages = 110 * 1024 / kStage < 2 ? 2 : 110 * 1024 / kStage > 4 ? 4 : 110 * 1024 / kStage;
    static constexpr int kSums = RT * 16 * kSortTokens;
    static constexpr int kRing = kStages * kStage > kSums * 8 ? kStages * kStage : kSums * 8;   // at the end: half of the warps' sums
    static constexpr int kSmem = kRing + kSums * 4;
};

__device__ __forceinline__ void lora_copy16(uint32_t dst, const void *src, bool ok) {  // zeros where not
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

__device__ __forceinline__ void lora_copy4x4(uint32_t dst, const char *src, int left) {  // four words, those from `left` on as zeros
#pragma unroll
    for (int j = 0; j < 4; ++j)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + j * 4), "l"(src + j * 4), "r"(j < left ? 4 : 0) : "memory");
}
__device__ __forceinline__ void lora_take8(uint32_t dst, const char *src, int left) {    // eight bf16, those from `left` on as zeros
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b16 l, h;\n\tmov.b16 l, 0;\n\tmov.b16 h, 0;\n\tsetp.gt.s32 p, %2, 0;\n\tsetp.gt.s32 q, %2, 1;\n\t"
                     "@p ld.global.nc.b16 l, [%1];\n\t@q ld.global.nc.b16 h, [%1+2];\n\tmov.b32 %0, {l, h};\n\t}"
                     : "=r"(w[j]) : "l"(src + j * 4), "r"(left - 2 * j) : "memory");
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// Into how many parts K of a tile is cut, as a power of two: as many as let all blocks run at once.  The tiles are known on
// the device alone: with the cut of all tiles that a table of 200 adapters can give, one request's 600 tokens at rank 64
// and K 8192 took 45 us, with that of its own 10 tiles 17; 600 tokens of 200 adapters 71 with either.
__host__ __device__ __forceinline__ int lora_shrink_cut(int tiles, int most, int at_once) {
    int cut = 0;
    while (cut < most && tiles <= at_once >> (cut + 1)) ++cut;
    return cut;
}
template <int RT, bool XF32, bool VEC>
constexpr int kShrinkBlocks = RT == 1 || (VEC && (RT == 2 || (RT == 4 && !XF32))) ? 2 : 1;   // an SM (registers)

// S = A x^T of a tile, K cut over blocks of a cluster, which holds as many tiles as the cut leaves room for.  Eight warps:
// two halves of the tokens, four steps of 32 of a stage's K.  Rows lie in shared memory as in global memory, their 16-byte
// pieces swapped by the row's last three bits so that the eight rows of a matrix lie in different banks.
// VEC: rows of x and A are 16-byte aligned.  Else their values are copied one by one, bf16 ones through registers.
template <int RT, bool XF32, bool VEC>
__global__ void __launch_bounds__(kLoraThreads, kShrinkBlocks<RT, XF32, VEC>) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
    namespace cg = cooperative_groups;
    using S = ShrinkShape<RT, XF32>;
    extern __shared__ __align__(128) uint8_t lora_smem[];
    float *const got = reinterpret_cast<float *>(lora_smem + S::kRing);   // [block][kSums / C]: this block's share of all blocks' sums
    __shared__ int32_t toks[kSortTokens];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3, kg = warp & 3, half = warp >> 2;
    cg::cluster_group cl = cg::this_cluster();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    const int own = 31 - __clz(p.cluster);
    LoraTile q = p.tiles[blockIdx.x >> own];            // (the tile if the cut is the cluster's, asked for beside the counts)
    const int count = p.tiles_count[0], served = p.tiles_count[1], cut = lora_shrink_cut(served, p.most, 148 * kShrinkBlocks<RT, XF32, VEC>);
    if ((cut == 0) != (own == 0)) return;               // the other launch's batch
    const int behind = (int)blockIdx.x - (served << cut);
    if (behind >= 0) {  // behind the tiles of an adapter, a block each, those of tokens without one
        if (served + behind >= count) return;
        q = p.tiles[served + behind];
        if (tid < kSortTokens) toks[tid] = tid < q.count ? p.perm[q.start + tid] : -1;
        __syncthreads();
        lora_none<true>(p, toks, kSortTokens, 0, 1);
        return;             // (a cluster's meetings do not wait for blocks that have left)
    }
    const int C = 1 << cut, part = blockIdx.x & (C - 1), rank0 = blockIdx.x & (p.cluster - 1) & -C;   // rank0: the tile's first block in the cluster
    if (cut != own) q = p.tiles[blockIdx.x >> cut];
    if (tid < kSortTokens) toks[tid] = tid < q.count ? p.perm[q.start + tid] : -1;
    __syncthreads();
    if (C > 1) cl.barrier_arrive();  // waited for before another block's shared memory is written
    // What this thread copies: one 16-byte column of every sixteenth row (of x in fp32: of every eighth).  Places without a
    // token and ranks behind the last one read the first's; nothing of them is stored.
    constexpr int XP = XF32 ? 32 : 16, XR = kLoraThreads / XP, XN = kSortTokens / XR, xe = XF32 ? 4 : 8;
    const int steps = (p.k + kSortK - 1) / kSortK, s0 = steps * part >> cut, s1 = steps * (part + 1) >> cut;
    const int xc = tid % XP, ac = tid % 16;
    const char *xsrc[XN], *asrc[RT];
#pragma unroll
    for (int i = 0; i < XN; ++i) {
        const int tok = toks[tid / XP + i * XR];
        xsrc[i] = static_cast<const char *>(p.x) + ((tok < 0 ? toks[0] : tok) * p.ldx + (int64_t)s0 * kSortK + xc * xe) * (XF32 ? 4 : 2);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int rank = tid / 16 + i * 16;
        asrc[i] = reinterpret_cast<const char *>(p.a + ((int64_t)q.adapter * p.r + (rank < p.r ? rank : 0)) * p.k + s0 * kSortK + ac * 8);
    }
    const uint32_t ring = smem_u32(lora_smem);
    // (a thread's rows are a multiple of eight apart: one swap for all)
    const uint32_t xdst = ring + tid / XP * (kSortK * (XF32 ? 4 : 2)) + (xc ^ (tid / XP & 7)) * 16;
    const uint32_t adst = ring + S::kX + tid / 16 * (kSortK * 2) + (ac ^ (tid / 16 & 7)) * 16;
    int slot_in = 0, slot_out = 0;
    auto request = [&](int st) {
        if (st < s1) {
            const bool whole = (st + 1) * kSortK <= p.k;
            const bool xin = whole || st * kSortK + xc * xe < p.k, ain = whole || st * kSortK + ac * 8 < p.k;
            const uint32_t at = slot_in * S::kStage;
#pragma unroll
            for (int i = 0; i < XN; ++i) {
                const uint32_t dst = xdst + at + i * XR * (kSortK * (XF32 ? 4 : 2));
                if (VEC) lora_copy16(dst, xsrc[i], xin);
                else if (XF32) lora_copy4x4(dst, xsrc[i], p.k - st * kSortK - xc * xe);
                else lora_take8(dst, xsrc[i], p.k - st * kSortK - xc * xe);
                xsrc[i] += kSortK * (XF32 ? 4 : 2);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (VEC) lora_copy16(adst + at + i * 16 * (kSortK * 2), asrc[i], ain);
                else lora_take8(adst + at + i * 16 * (kSortK * 2), asrc[i], p.k - st * kSortK - ac * 8);
                asrc[i] += kSortK * 2;
            }
        }
        slot_in = slot_in + 1 == S::kStages ? 0 : slot_in + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i + 1 < S::kStages; ++i) request(s0 + i);
    float acc[RT][4][4] = {};
    for (int st = s0; st < s1; ++st) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        __syncthreads();  // the stage is there for all, and the one before it is read by all
        request(st + S::kStages - 1);
        const uint8_t *const xs = lora_smem + slot_out * S::kStage, *const as = xs + S::kX;
        slot_out = slot_out + 1 == S::kStages ? 0 : slot_out + 1;
        uint4 aw[RT][2];
        const uint32_t xa = smem_u32(xs), aa = smem_u32(as);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)  // ranks 0-7, 8-15 of K 0-7, then of K 8-15
                ldmatrix_x4(aa + (i * 16 + (lane & 15)) * (kSortK * 2) + ((kg * 4 + h * 2 + (lane >> 4)) ^ (lane & 7)) * 16, aw[i][h].x, aw[i][h].y, aw[i][h].z, aw[i][h].w);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            float f[8];
            uint4 xv;
            if (XF32) {
                const uint8_t *r = xs + (half * 32 + n * 8 + g) * (kSortK * 4) + (t4 & 1) * 8;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<float2 *>(f + 2 * j) = *reinterpret_cast<const float2 *>(r + ((kg * 8 + j * 2 + (t4 >> 1)) ^ g) * 16);
            } else {  // K 0-7, 8-15, 16-23, 24-31 of eight tokens
                ldmatrix_x4(xa + (half * 32 + n * 8 + (lane & 7)) * (kSortK * 2) + ((kg * 4 + (lane >> 3)) ^ (lane & 7)) * 16, xv.x, xv.y, xv.z, xv.w);
            }
#pragma unroll
            for (int w = 0; w < (XF32 ? 3 : 1); ++w) {
                if (XF32) xv = make_uint4(cut_bf16x2(f[0], f[1]), cut_bf16x2(f[2], f[3]), cut_bf16x2(f[4], f[5]), cut_bf16x2(f[6], f[7]));
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    mma_bf16(acc[i][n], aw[i][0].x, aw[i][0].y, aw[i][0].z, aw[i][0].w, xv.x, xv.y);
                    mma_bf16(acc[i][n], aw[i][1].x, aw[i][1].y, aw[i][1].z, aw[i][1].w, xv.z, xv.w);
                }
            }
        }
    }
    // the four steps' sums: 2 and 3 to 0 and 1, then 1 to 0
    float *const sums = reinterpret_cast<float *>(lora_smem);
    constexpr int kMine = RT * 4 * 128;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int from = 2; from; from >>= 1) {
        __syncthreads();
        float *const at = sums + ((kg % from) * 2 + half) * kMine + lane;
        if (kg >= from && kg < 2 * from)
#pragma unroll
            for (int j = 0; j < RT * 16; ++j) at[j * 32] = acc[j / 16][j / 4 % 4][j % 4];
        __syncthreads();
        if (kg < from)
#pragma unroll
            for (int j = 0; j < RT * 16; ++j) acc[j / 16][j / 4 % 4][j % 4] += at[j * 32];
    }
    // every block of the cluster adds one share of the sums up
    const int share = S::kSums >> cut;
    if (C > 1) cl.barrier_wait();
    if (kg == 0)
#pragma unroll
        for (int j = 0; j < RT * 16; ++j) {
            const int at = half * kMine + j * 32 + lane, c = at / share;
            (C > 1 ? cl.map_shared_rank(got, rank0 + c) : got)[part * share + at - c * share] = acc[j / 16][j / 4 % 4][j % 4];
        }
    if (C > 1) cl.sync();
    else __syncthreads();
    for (int j = tid; j < share; j += kLoraThreads) {
        float s = 0.0f;
        for (int c = 0; c < C; ++c) s += got[c * share + j];
        const int at = part * share + j, l = at & 31, e = at >> 5 & 3, n = at >> 7 & 3, i = (at % kMine) >> 9, h = at / kMine;
        const int rank = i * 16 + (l >> 2) + (e >> 1) * 8, tok = toks[h * 32 + n * 8 + (l & 3) * 2 + (e & 1)];
        if (tok >= 0 && rank < p.r) p.s_out[(int64_t)tok * p.r + rank] = s;
    }
}

// out = y + B S of a tile and a slice of N, 64 rows of B a warp at a time.  Here the tokens are the rows of the product
// and B's rows its columns: a fragment of B is two neighbouring registers of a 16-byte load, and S lies in shared memory
// in fragments, so nothing is moved between registers (with the operands the other way round, four moves a product,
// 73 us for the 4000 rows of rank 64).  Row 16 q + 4 (c / 2) + 2 i + c % 2 of the 64 is column c of product 2 q + i,
// which leaves a lane four consecutive outputs of a token.  The y of a step, 16 tokens and 32 rows of B, is requested
// kAhead steps ahead of its sum: four where registers allow it (rank 64, 4000 rows of 7168 66.6 us, with two 67.4), else two
// (the others spill more with four: rank 16 53 us against 70, rank 32 74 against 87, rank 128 144 against 171).
template <int RT>
struct ExpandShape {
    static constexpr int kFragments = 4 * RT;                     // (tokens of 16, ranks of 16)
    static constexpr int kSmem = 3 * kFragments * 512;
};
constexpr int kExpandN = kLoraWarps * 64;     // rows of B a block takes at a time

// VEC: four consecutive values of y and of out are one access.
template <int RT, bool YF32, bool VEC>
__global__ void __launch_bounds__(kLoraThreads, RT <= 2 ? 2 : 1) lora_expand_kernel(const __grid_constant__ LoraParams p) {
    using S = ExpandShape<RT>;
    constexpr int es = YF32 ? 4 : 2, kStepsN = kSortTokens / 16 * 2, kAhead = RT == 4 ? 4 : 2;
    extern __shared__ __align__(128) uint8_t lora_smem[];
    __shared__ int32_t toks[kSortTokens];
    __shared__ int64_t yoff[kSortTokens], ooff[kSortTokens];    // bytes; places without a token read the first one's
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int slices = p.cluster, slice = blockIdx.x % slices, tile = blockIdx.x / slices;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    wait_predecessor();
    if (tile >= *p.tiles_count) return;
    const LoraTile q = p.tiles[tile];
    if (tid < kSortTokens) {
        const int tok = p.perm[q.start + (tid < q.count ? tid : 0)];
        toks[tid] = tid < q.count ? tok : -1;
        yoff[tid] = tok * p.ldy * es;
        ooff[tid] = tok * p.ldo * es;
    }
    __syncthreads();
    if (q.adapter < 0) {
        lora_none<VEC>(p, toks, kSortTokens, slice, slices);
        return;
    }
    constexpr int KP = RT >= 2 ? RT / 2 : 1;
    const int rounds = (p.n + kExpandN - 1) / kExpandN, r0 = (int)((int64_t)rounds * slice / slices), r1 = (int)((int64_t)rounds * (slice + 1) / slices);
    const uint16_t *const table = p.b + (int64_t)q.adapter * p.n * p.r;
    uint4 bw[8][KP];
    auto weights = [&](int n0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = n0 + (j >> 1) * 16 + (g >> 1) * 4 + (j & 1) * 2 + (g & 1);
            const uint16_t *b = table + (int64_t)min(row, p.n - 1) * p.r;
            if (RT >= 2) {
#pragma unroll
                for (int k = 0; k < KP; ++k) bw[j][k] = row8<true>(b, k * 32 + t4 * 8, p.r);
            } else {
                const uint2 v = load8_if(b + t4 * 4, t4 * 4 < p.r);
                bw[j][0] = make_uint4(v.x, v.y, 0, 0);
            }
        }
    };
    const char *const ybase = static_cast<const char *>(p.y);
    char *const obase = static_cast<char *>(p.out);
    uint4 yv[kAhead][4];
    auto request = [&](int s, int n0) {  // (rows behind the last one's read that; nothing of them is stored)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int nn = n0 + ((s & 1) * 2 + (e & 1)) * 16 + t4 * 4;
            const char *row = ybase + yoff[(s >> 1) * 16 + (e >> 1) * 8 + g];
            uint4 &r = yv[s % kAhead][e];
            // (y may be out: not a read-only load)
            if (VEC) {
                const char *src = row + min(nn, p.n - 4) * es;
                if (YF32) asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(src) : "memory");
                else asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(src) : "memory");
            } else {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const char *src = row + min(nn + j, p.n - 1) * es;
                    if (YF32) asm volatile("ld.global.b32 %0, [%1];" : "=r"(v[j]) : "l"(src) : "memory");
                    else asm volatile("{\n\t.reg .b16 h, z;\n\tmov.b16 z, 0;\n\tld.global.b16 h, [%1];\n\tmov.b32 %0, {z, h};\n\t}" : "=r"(v[j]) : "l"(src) : "memory");
                }
                r = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
    };
    weights(r0 * kExpandN + warp * 64);
#pragma unroll
    for (int s = 0; s < kAhead; ++s) request(s, r0 * kExpandN + warp * 64);
    // scale * S in three bf16 parts, as fragments: ranks of a lane as B's 16-byte loads have them
    const float scale = p.scale ? p.scale[q.adapter] : 1.0f;
    for (int j = tid; j < kSortTokens * RT * 8; j += kLoraThreads) {
        const int place = j / (RT * 8), rank = j % (RT * 8) * 2, tok = toks[place];
        float2 s = make_float2(0.0f, 0.0f);
        if (tok >= 0 && rank < p.r) {  // (r is even; the shrunk rows may be a caller's, aligned to 4 bytes: no vector)
            const float *const src = p.s_in + (int64_t)tok * p.r + rank;
            s = make_float2(src[0], src[1]);
        }
        s.x *= scale;
        s.y *= scale;
        const int step = RT >= 2 ? rank / 32 * 2 + rank % 8 / 4 : 0, col = RT >= 2 ? rank % 32 / 8 : rank / 4;
        const int at = (place / 16 * RT + step) * 512 + (place % 8 * 4 + col) * 16 + (rank % 4 / 2 * 2 + place % 16 / 8) * 4;
#pragma unroll
        for (int w = 0; w < 3; ++w) *reinterpret_cast<uint32_t *>(lora_smem + w * S::kFragments * 512 + at) = cut_bf16x2(s.x, s.y);
    }
    __syncthreads();
    for (int r = r0; r < r1; ++r) {
        const int n0 = r * kExpandN + warp * 64;
#pragma unroll
        for (int s = 0; s < kStepsN; ++s) {
            float acc[4][4] = {};
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    const uint4 f = *reinterpret_cast<const uint4 *>(lora_smem + ((w * 4 + (s >> 1)) * RT + k) * 512 + lane * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 &b = bw[(s & 1) * 4 + j][k / 2];
                        mma_bf16(acc[j], f.x, f.y, f.z, f.w, k & 1 ? b.z : b.x, k & 1 ? b.w : b.y);
                    }
                }
            // the next rows of B while the last sums of these are stored
            if (s == kStepsN - 1 && r + 1 < r1) weights(n0 + kExpandN);
            float sum[4][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint4 &y = yv[s % kAhead][e];
                const int j = (e & 1) * 2, h = (e >> 1) * 2;
                constexpr bool packed = VEC && !YF32;
                sum[e][0] = __uint_as_float(packed ? y.x << 16 : y.x) + acc[j][h];
                sum[e][1] = __uint_as_float(packed ? y.x & 0xFFFF0000u : y.y) + acc[j][h + 1];
                sum[e][2] = __uint_as_float(packed ? y.y << 16 : y.z) + acc[j + 1][h];
                sum[e][3] = __uint_as_float(packed ? y.y & 0xFFFF0000u : y.w) + acc[j + 1][h + 1];
            }
            if (s + kAhead < kStepsN) request(s + kAhead, n0);
            else if (r + 1 < r1) request(s + kAhead - kStepsN, n0 + kExpandN);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int place = (s >> 1) * 16 + (e >> 1) * 8 + g, nn = n0 + ((s & 1) * 2 + (e & 1)) * 16 + t4 * 4;
                if (place >= q.count || nn >= p.n) continue;
                char *const dst = obase + ooff[place] + (int64_t)nn * es;
                if (!VEC) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (nn + i < p.n) store1(dst, YF32 ? WS_ACT_F32 : WS_ACT_BF16, i, sum[e][i]);
                } else if (YF32) *reinterpret_cast<float4 *>(dst) = make_float4(sum[e][0], sum[e][1], sum[e][2], sum[e][3]);
                else *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(sum[e][0], sum[e][1]), pack_bf16x2(sum[e][2], sum[e][3]));
            }
        }
    }
}

}  // namespace ws
