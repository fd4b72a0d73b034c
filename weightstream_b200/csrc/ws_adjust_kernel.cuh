// Bias, penalties for repeated tokens and grammar masks on a row of logits:
//
//   z = x + bias[v]                                     (of the row's listed tokens; the last entry of a token counts)
//   z = z > 0 ? z / r : z * r                           where v occurs in the row's history
//   z = z - f * count - p * (count > 0)                 count: occurrences behind the history's first `prompt` tokens
//   z = -inf                                            where the row's mask has no bit for v
//
// A block takes a slice of a row's vocabulary that fits its registers: it requests its logits first, counts the row's
// history into a table of its slice in shared memory while they come, and writes every value once.  So a row's history
// is read by each of its blocks (out of L2), and nothing is exchanged between them.
#pragma once

#include "ws_values.cuh"

namespace ws {

constexpr int kAdjustThreads = 256;
constexpr uint32_t kAdjustPrompt = 0x80000000u;    // a table's word: occurrences in the answer, this bit for one in the prompt

struct AdjustParams {
    const void *logits;
    void *out;
    int64_t ld, ldo;
    const int32_t *tokens;                          // histories of all rows, one after the other; null: none
    const void *offsets;                            // [m + 1] into tokens
    const int32_t *prompt_lens;                     // [m] or null: 0
    const float *repetition, *frequency, *presence; // [m] or null: 1, 0, 0
    const int32_t *bias_ids;
    const float *bias;
    const void *bias_offsets;                       // [m + 1] into bias
    const uint32_t *mask;                           // [mask_count, ld_mask] words, bit v % 32 of word v / 32: v is allowed
    const int32_t *mask_rows;                       // [m] or null: row t of the mask
    int64_t n_tokens, n_bias, ld_mask;
    int32_t m, vocab, mask_count, offset_bytes, bias_offset_bytes, slices;
};

// Bounds of a row's entries, whatever the offsets hold.
__device__ __forceinline__ void adjust_range(const void *offsets, int bytes, int t, int64_t n, int64_t &a, int64_t &b) {
    if (bytes == 8) { a = static_cast<const int64_t *>(offsets)[t]; b = static_cast<const int64_t *>(offsets)[t + 1]; }
    else { a = static_cast<const int32_t *>(offsets)[t]; b = static_cast<const int32_t *>(offsets)[t + 1]; }
    a = a < 0 ? 0 : a > n ? n : a;
    b = b < a ? a : b > n ? n : b;
}

struct AdjustRow {
    float rep, freq, pres;
    bool masked;
    const uint32_t *mask;
};

__device__ __forceinline__ float adjust_value(float z, uint32_t word, const AdjustRow &r) {
    if (word) {
        z = z > 0.0f ? __fdiv_rn(z, r.rep) : z * r.rep;
        const uint32_t n = word & ~kAdjustPrompt;
        if (n) z = fmaf(-r.freq, (float)n, z) - r.pres;
    }
    return z;
}

// VEC: rows are read and written 16 bytes at a time.  A row's values lie on a grid of vectors that begins at its first
// aligned address or one vector before; values of the first and last vector that are not the row's are left alone.
template <bool F32, bool VEC, int U>
__global__ void __launch_bounds__(kAdjustThreads) adjust_kernel(const __grid_constant__ AdjustParams p) {
    constexpr int W = F32 ? 4 : 8;                  // values a vector
    constexpr int kSlice = kAdjustThreads * U * W;
    extern __shared__ uint32_t adjust_table[];      // counts, then places of biases (1 + entry), as far as the call has them
    uint32_t *const count_s = adjust_table, *const bias_s = adjust_table + (p.tokens ? kSlice : 0);
    const int t = blockIdx.x / p.slices, slice = blockIdx.x % p.slices, tid = threadIdx.x;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const char *const x = static_cast<const char *>(p.logits) + (int64_t)t * p.ld * (F32 ? 4 : 2);
    char *const y = static_cast<char *>(p.out) + (int64_t)t * p.ldo * (F32 ? 4 : 2);
    const int skew = VEC ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / (F32 ? 4 : 2)) : 0;  // the grid begins so many values before the row
    const int v0 = slice * kSlice - skew;
    for (int i = tid * 4; i < (p.tokens ? kSlice : 0) + (p.bias_ids ? kSlice : 0); i += kAdjustThreads * 4)
        *reinterpret_cast<uint4 *>(adjust_table + i) = make_uint4(0u, 0u, 0u, 0u);
    wait_predecessor();
    // ---- the slice's logits
    uint32_t raw[U][4];
    if constexpr (VEC) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + (u * kAdjustThreads + tid) * W;
            raw[u][0] = raw[u][1] = raw[u][2] = raw[u][3] = 0u;
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                         : "+r"(raw[u][0]), "+r"(raw[u][1]), "+r"(raw[u][2]), "+r"(raw[u][3])
                         : "l"(x + (int64_t)v * (F32 ? 4 : 2)), "r"((int)(v >= 0 && v <= p.vocab - W)) : "memory");
        }
    }
    AdjustRow r;
    r.rep = p.repetition ? p.repetition[t] : 1.0f;
    r.freq = p.frequency ? p.frequency[t] : 0.0f;
    r.pres = p.presence ? p.presence[t] : 0.0f;
    int which = -1;
    if (p.mask) which = p.mask_rows ? p.mask_rows[t] : t;
    r.masked = which >= 0 && which < p.mask_count;
    r.mask = p.mask + (r.masked ? which * p.ld_mask : 0);
    __syncthreads();
    // ---- the row's history and biases that fall into the slice
    if (p.tokens) {
        int64_t a, b;
        adjust_range(p.offsets, p.offset_bytes, t, p.n_tokens, a, b);
        const int64_t prompt = a + (p.prompt_lens ? p.prompt_lens[t] : 0);
        for (int64_t i = a + tid; i < b; i += kAdjustThreads) {
            const int32_t v = p.tokens[i];
            const uint32_t at = (uint32_t)(v - v0);
            if (v >= 0 && v < p.vocab && at < (uint32_t)kSlice) {
                if (i < prompt) atomicOr(&count_s[at], kAdjustPrompt);
                else atomicAdd(&count_s[at], 1u);
            }
        }
    }
    if (p.bias_ids) {
        int64_t a, b;
        adjust_range(p.bias_offsets, p.bias_offset_bytes, t, p.n_bias, a, b);
        for (int64_t i = a + tid; i < b; i += kAdjustThreads) {
            const int32_t v = p.bias_ids[i];
            const uint32_t at = (uint32_t)(v - v0);
            if (v >= 0 && v < p.vocab && at < (uint32_t)kSlice) atomicMax(&bias_s[at], (uint32_t)(i - a) + 1u);
        }
    }
    int64_t bias0 = 0, bias1;
    if (p.bias_ids) adjust_range(p.bias_offsets, p.bias_offset_bytes, t, p.n_bias, bias0, bias1);
    __syncthreads();
    auto one = [&](float z, int at, int v) {
        if (p.bias_ids) {
            const uint32_t e = bias_s[at];
            if (e) z += p.bias[bias0 + e - 1];
        }
        if (p.tokens) z = adjust_value(z, count_s[at], r);
        if (r.masked && !(r.mask[v >> 5] >> (v & 31) & 1u)) z = __uint_as_float(0xFF800000u);
        return z;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int at = (u * kAdjustThreads + tid) * W, v = v0 + at;
        if (VEC && v >= 0 && v <= p.vocab - W) {
            float z[W];
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const uint32_t w = raw[u][F32 ? e & 3 : e / 2];
                z[e] = one(__uint_as_float(F32 ? w : e & 1 ? w & 0xFFFF0000u : w << 16), at + e, v + e);
            }
            uint4 o;
            if constexpr (F32) o = make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
            else o = make_uint4(pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]), pack_bf16x2(z[4], z[5]), pack_bf16x2(z[6], z[7]));
            *reinterpret_cast<uint4 *>(y + (int64_t)v * (F32 ? 4 : 2)) = o;
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                // (values of a vector are a block apart where rows are read one by one)
                const int place = VEC ? at + e : (u * W + e) * kAdjustThreads + tid, w = v0 + place;
                if (w >= 0 && w < p.vocab) store1(y, F32 ? WS_ACT_F32 : WS_ACT_BF16, w, one(load1(x, F32 ? WS_ACT_F32 : WS_ACT_BF16, w), place, w));
            }
        }
    }
}

}  // namespace ws
