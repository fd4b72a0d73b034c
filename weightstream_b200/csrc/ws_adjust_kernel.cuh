// Bias, penalties for repeated tokens and grammar masks on a row of logits:
//
//   z = x + bias[v]                                     (of the row's listed tokens; the last entry of a token counts)
//   z = z > 0 ? z / r : z * r                           where v occurs in the row's history
//   z = z - f * count - p * (count > 0)                 count: occurrences behind the history's first `prompt` tokens
//   z = -inf                                            where the row's mask has no bit for v
//
// A block takes a slice of a row's vocabulary that fits its registers.  It requests its logits, counts the row's lists into a
// table of its slice in shared memory while they come (a row's lists are read by each of its blocks, out of L2; nothing is
// exchanged between blocks), stores the logits under the mask, and then takes the touched values by themselves: every
// thread notes which of its places are touched, and the block's threads share them out.
//
// Other ways, us for one row with 6000 tokens, 64 rows with 4000, 512 bf16 rows with 2000 under masks: touched values where they
// pass (most vectors of a warp have one, and all lanes wait for it) 6, 35 and 127; noted by who counts first 10, 29 and 86;
// clusters of a row's slices that count into each other's tables 19, 52 and 169; a plain copy, and a hash table a row beside
// or behind it 12, 33 and 91.
//
// Bound: instructions.  One row of 129280 with 6000 tokens 6.2 to 7.1 us, 64 rows with 4000, a mask and biases 26 to 27 us (10.3 of HBM),
// 512 bf16 rows with 2000 and masks 83 to 85 us (41; one call after the other 83 to 84, without lists 43, with lists of -1 69): a block's fixed part,
// the lists that each of a row's sixteen blocks looks through, and the mask's bits.
#pragma once

#include "ws_values.cuh"

namespace ws {

constexpr int kAdjustThreads = 256;
constexpr int kAdjustList = 2048;                   // touched places that are noted; beyond, the table is looked through
// A word of the table: 31 a bias; 30 to 16 occurrences in the prompt; 15 to 0 occurrences behind it.  Rows with longer
// histories: 30 an occurrence in the prompt, 29 to 0 occurrences behind it.
constexpr uint32_t kAdjustListed = 0x80000000u, kAdjustPrompt = 0x40000000u;
constexpr int kAdjustShort = 32767;
// Lists of biases are looked through for each of a row's listed values up to this length, on average over the batch; longer ones
// have their places in a table.  Lists of 32, 64 and 128 in all rows, us, looked through / in a second table: 64 fp32 rows 15.2 / 15.2, 19.3 / 15.6
// and 28 / 15.6, 512 bf16 rows with 2000 tokens each 91 / 118, 114 / 120 and 166 / 122.
constexpr int kAdjustFew = 64;
// The same for a row's own list in a batch of shorter ones, which costs more: it is gone through twice, with the row's tokens.  Every
// fourth row with a list of 128, 192 or 250, looked through / in halves: 64 fp32 rows 18.2 / 13.7, 22.5 / 14.3 and 26.5 / 14.6 us,
// 512 bf16 rows with 2000 tokens each 102 / 116, 121 / 118 and 142 / 119.
constexpr int kAdjustLong = 192;

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
    int32_t m, vocab, mask_count, offset_bytes, bias_offset_bytes, slices, in_place, bias_table;   // bias_table: a second table, of the biases' places
};

// Bounds of a row's entries, whatever the offsets hold.
__device__ __forceinline__ void adjust_range(const void *offsets, int bytes, int t, int64_t n, int64_t &a, int64_t &b) {
    if (bytes == 8) { a = static_cast<const int64_t *>(offsets)[t]; b = static_cast<const int64_t *>(offsets)[t + 1]; }
    else { a = static_cast<const int32_t *>(offsets)[t]; b = static_cast<const int32_t *>(offsets)[t + 1]; }
    a = a < 0 ? 0 : a > n ? n : a;
    b = b < a ? a : b > n ? n : b;
}

// f(entry, value) for the entries [a, b) of a list, by all threads of the block, four loads ahead.  (One copy of f: vectors of
// entries and a loop unrolled over them made 36 copies of it: one row with 6000 tokens took 36 us in an
// early form, with one copy 28.)
template <typename F>
__device__ __forceinline__ void adjust_list(const int32_t *list, int64_t a, int64_t b, F f) {
    const int step = blockDim.x;
    const int n = (int)min(b - a, (int64_t)INT32_MAX - 8 * 1024);       // (a row's own entries)
    const int32_t *const own = list + a;
    int32_t ahead[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) ahead[k] = (int)threadIdx.x + k * step < n ? own[threadIdx.x + k * step] : -1;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += step) {
        const int32_t v = ahead[0];
        ahead[0] = ahead[1];
        ahead[1] = ahead[2];
        ahead[2] = ahead[3];
        ahead[3] = i + 4 * step < n ? own[i + 4 * step] : -1;
        f(a + i, v);
    }
}

// f(place in the list, value) for its n entries, by all threads of the block: 16 bytes a load, two of them at once (four
// cost 2000 tokens as many instructions as 4000).
template <typename F>
__device__ __forceinline__ void adjust_tokens(const int32_t *list, int n, F f) {
    const int tid = threadIdx.x, head = min(n, (int)(16 - (reinterpret_cast<uintptr_t>(list) & 15)) / 4 & 3), vectors = (n - head) / 4;
    const int4 *const v = reinterpret_cast<const int4 *>(list + head);
#pragma unroll 1
    for (int i = tid; i < vectors; i += 2 * kAdjustThreads) {
        int4 t[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) t[k] = i + k * kAdjustThreads < vectors ? v[i + k * kAdjustThreads] : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = head + (i + k * kAdjustThreads) * 4;
            f(at, t[k].x);
            f(at + 1, t[k].y);
            f(at + 2, t[k].z);
            f(at + 3, t[k].w);
        }
    }
    const int ends = n - vectors * 4;               // before the first vector and behind the last
    if (tid < ends) {
        const int at = tid < head ? tid : tid + vectors * 4;
        f(at, list[at]);
    }
}

__device__ __forceinline__ const uint32_t *adjust_mask(const AdjustParams &p, int t) {    // null: none
    const int which = !p.mask ? -1 : p.mask_rows ? p.mask_rows[t] : t;
    return which >= 0 && which < p.mask_count ? p.mask + which * p.ld_mask : nullptr;
}
__device__ __forceinline__ bool adjust_open(const uint32_t *mask, int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1u); }
constexpr uint32_t kAdjustMinusInf = 0xFF800000u;

// A word of logits under the first bits of a mask.
template <bool F32>
__device__ __forceinline__ void adjust_close(uint32_t &w, uint32_t bits) {
    if constexpr (F32) {
        w = bits & 1u ? w : kAdjustMinusInf;
    } else {
        const uint32_t keep = ((bits & 3u) * 0x8001u & 0x10001u) * 0xFFFFu;        // two bits to two halves
        w = (w & keep) | (0xFF80FF80u & ~keep);
    }
}

// A row of a block: its lists, its mask, where its slice begins.
struct AdjustRow {
    const AdjustParams &p;
    int t, v0;                                      // v0: the token of the slice's first place
    int64_t a, b, bias0, bias1;

    __device__ __forceinline__ AdjustRow(const AdjustParams &p, int t, int v0) : p(p), t(t), v0(v0), a(0), b(0), bias0(0), bias1(0) {
        if (p.tokens) adjust_range(p.offsets, p.offset_bytes, t, p.n_tokens, a, b);
        if (p.bias_ids) adjust_range(p.bias_offsets, p.bias_offset_bytes, t, p.n_bias, bias0, bias1);
    }
    __device__ __forceinline__ bool packed() const { return b - a <= kAdjustShort; }    // (the block's conditions)
    // Counts the lists' tokens of `span` places from `from` on into the table, and with `last` the places of biases from that
    // word of it on.
    __device__ __forceinline__ void count(uint32_t *table, int from, int span, int last) const {
        const int low = max(v0 + from, 0);          // those tokens: low and `width` behind it
        const uint32_t width = (uint32_t)max(0, min(v0 + from + span, p.vocab) - low);
        uint32_t *const word = table + (low - v0 - from);
        if (bias1 > bias0)
            adjust_list(p.bias_ids, bias0, bias1, [&](int64_t i, int32_t v) {
                if ((uint32_t)(v - low) >= width) return;
                atomicOr(&word[v - low], kAdjustListed);
                if (last) atomicMax(&word[v - low + last], (uint32_t)(i - bias0) + 1u);
            });
        if (b > a) {
            const int behind_at = p.prompt_lens ? p.prompt_lens[t] : 0;
            const int64_t prompt = a + behind_at;
            if (packed())
                adjust_tokens(p.tokens + a, (int)(b - a), [&](int i, int32_t v) {
                    if ((uint32_t)(v - low) < width) atomicAdd(&word[v - low], i < behind_at ? 0x10000u : 1u);
                });
            else
                adjust_list(p.tokens, a, b, [&](int64_t i, int32_t v) {
                    if ((uint32_t)(v - low) >= width) return;
                    if (i < prompt) atomicOr(&word[v - low], kAdjustPrompt);
                    else atomicAdd(&word[v - low], 1u);
                });
        }
    }
    // What becomes of the value of token v, whose word of the table is `word`; `listed`: its bias' place and one more, 0 where
    // that is still to be looked for.
    __device__ __forceinline__ void change(const char *x, char *y, int type, int v, uint32_t word, uint32_t listed, float rep, float freq, float pres) const {
        float z = load1(x, type, v);
        if (word & kAdjustListed) {                 // its last entry
            int64_t e = bias0 + listed;
            if (!listed)
                for (e = bias1; e > bias0 && p.bias_ids[e - 1] != v;) --e;
            if (e > bias0) z += p.bias[e - 1];
        }
        const uint32_t behind = packed() ? word & 0xFFFFu : word & (kAdjustPrompt - 1u);
        if (word & ~kAdjustListed) z = z > 0.0f ? __fdiv_rn(z, rep) : z * rep;
        if (behind) z = fmaf(-freq, (float)behind, z) - pres;
        store1(y, type, v, z);
    }
    __device__ __forceinline__ float of(const float *values, float otherwise) const { return values && b > a ? values[t] : otherwise; }
};

// The touched values of a slice whose row has a long list of biases in a batch of short ones, after its logits have been
// stored: in halves, so that the table's second half has room for the places of the first one's biases.  Every place of the table is
// looked at.  (A function of its own: as a branch of the kernel it cost all other rows 2 to 6 %.)
template <bool F32, int SLICE>
__device__ __noinline__ void adjust_halves(const AdjustParams &p, uint32_t *table, int t, int v0) {
    const AdjustRow r(p, t, v0);
    const uint32_t *const mask = adjust_mask(p, t);
    const char *const x = static_cast<const char *>(p.logits) + (int64_t)t * p.ld * (F32 ? 4 : 2);
    char *const y = static_cast<char *>(p.out) + (int64_t)t * p.ldo * (F32 ? 4 : 2);
    const float rep = r.of(p.repetition, 1.0f), freq = r.of(p.frequency, 0.0f), pres = r.of(p.presence, 0.0f);
#pragma unroll 1
    for (int from = 0; from < SLICE; from += SLICE / 2) {
        if (from) {
            __syncthreads();                        // the first half's values have been taken
#pragma unroll 1
            for (int i = threadIdx.x; i < SLICE; i += kAdjustThreads) table[i] = 0u;
        }
        __syncthreads();
        r.count(table, from, SLICE / 2, SLICE / 2);
        __syncthreads();
#pragma unroll 1
        for (int at = threadIdx.x; at < SLICE / 2; at += kAdjustThreads) {
            const uint32_t word = table[at];
            if (word && adjust_open(mask, v0 + from + at)) r.change(x, y, F32 ? WS_ACT_F32 : WS_ACT_BF16, v0 + from + at, word, table[at + SLICE / 2], rep, freq, pres);
        }
    }
}

// VEC: rows are read and written 16 bytes at a time.  A row's values lie on a grid of vectors that begins at its first
// aligned address or one vector before; values of the first and last vector that are not the row's are left alone.
template <bool F32, bool VEC, int U, int BLOCKS>
__global__ void __launch_bounds__(kAdjustThreads, BLOCKS) adjust_kernel(const __grid_constant__ AdjustParams p) {
    constexpr int W = F32 ? 4 : 8, kType = F32 ? WS_ACT_F32 : WS_ACT_BF16;      // values a vector
    constexpr int kSlice = kAdjustThreads * U * W;
    static_assert(U * W <= 64 && kSlice <= 65536, "a bit for each of a thread's places; a place is 16 bits");
    extern __shared__ __align__(16) uint32_t adjust_table[];
    __shared__ uint16_t list_s[kAdjustList];
    __shared__ int touched_s;
    const int t = blockIdx.x / p.slices, slice = blockIdx.x - t * p.slices, tid = threadIdx.x, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const char *const x = static_cast<const char *>(p.logits) + (int64_t)t * p.ld * (F32 ? 4 : 2);
    char *const y = static_cast<char *>(p.out) + (int64_t)t * p.ldo * (F32 ? 4 : 2);
    const int skew = VEC ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / (F32 ? 4 : 2)) : 0;  // the grid begins so many values before the row
    const int v0 = slice * kSlice - skew;
    const bool lists = p.tokens || p.bias_ids;
    if (lists) {
#pragma unroll 1
        for (int i = tid * 4; i < (p.bias_table ? 2 * kSlice : kSlice); i += kAdjustThreads * 4) *reinterpret_cast<uint4 *>(adjust_table + i) = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) touched_s = 0;
    }
    wait_predecessor();
    // ---- what the row's lists are, then the slice's logits, then the lists
    const AdjustRow r(p, t, v0);
    const uint32_t *const mask = adjust_mask(p, t);
    const bool dense = mask || !p.in_place;         // (else only touched values change)
    uint32_t raw[U][4];
    if constexpr (VEC) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + (u * kAdjustThreads + tid) * W;
            raw[u][0] = raw[u][1] = raw[u][2] = raw[u][3] = 0u;
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                         : "+r"(raw[u][0]), "+r"(raw[u][1]), "+r"(raw[u][2]), "+r"(raw[u][3])
                         : "l"(x + (int64_t)v * (F32 ? 4 : 2)), "r"((int)(dense && v >= 0 && v <= p.vocab - W)) : "memory");
        }
    }
    const bool listed = r.bias1 > r.bias0 || r.b > r.a, halves = !p.bias_table && r.bias1 - r.bias0 > kAdjustLong;   // (the block's conditions)
    if (listed && !halves) {
        __syncthreads();
        r.count(adjust_table, 0, kSlice, p.bias_table ? kSlice : 0);
    }
    // ---- the logits under the mask
    if (dense) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (u * kAdjustThreads + tid) * W, v = v0 + at;
            if (VEC && v >= 0 && v <= p.vocab - W) {
                if (mask) {                         // (a vector of a row that is not aligned may lie in two words)
                    const uint32_t bits = __funnelshift_r(mask[v >> 5], mask[(v + W - 1) >> 5], v & 31);
#pragma unroll
                    for (int k = 0; k < 4; ++k) adjust_close<F32>(raw[u][k], bits >> (F32 ? k : 2 * k));
                }
                *reinterpret_cast<uint4 *>(y + (int64_t)v * (F32 ? 4 : 2)) = make_uint4(raw[u][0], raw[u][1], raw[u][2], raw[u][3]);
            } else {
#pragma unroll 1
                for (int k = 0; k < W; ++k) {
                    // (values of a vector are a block apart where rows are read one by one)
                    const int w = v0 + (VEC ? at + k : (u * W + k) * kAdjustThreads + tid);
                    if (w < 0 || w >= p.vocab) continue;
                    const float z = load1(x, kType, w);
                    store1(y, kType, w, adjust_open(mask, w) ? z : __uint_as_float(kAdjustMinusInf));
                }
            }
        }
    }
    if (!listed) return;
    if (halves) return adjust_halves<F32, kSlice>(p, adjust_table, t, v0);
    // ---- the touched places, a bit each of this thread's
    __syncthreads();
    uint64_t mine = 0u;
#pragma unroll
    for (int q = 0; q < U * W / 4; ++q) {
        const uint4 w = *reinterpret_cast<const uint4 *>(adjust_table + (q * kAdjustThreads + tid) * 4);
        if (w.x | w.y | w.z | w.w) mine |= (uint64_t)((w.x ? 1u : 0u) | (w.y ? 2u : 0u) | (w.z ? 4u : 0u) | (w.w ? 8u : 0u)) << 4 * q;
    }
    const int count = __popcll(mine);
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
    }
    int place = 0;
    if (lane == 31 && upto) place = atomicAdd(&touched_s, upto);
    place = __shfl_sync(0xffffffffu, place, 31) + upto - count;
    for (uint64_t left = mine; left; left &= left - 1, ++place) {
        const int bit = __ffsll(left) - 1;
        if (place < kAdjustList) list_s[place] = (uint16_t)(((bit >> 2) * kAdjustThreads + tid) * 4 + (bit & 3));
    }
    __syncthreads();
    // ---- their values.  (In place the mask has been at x already, which gives the same.)
    const int touched = touched_s, all = touched <= kAdjustList ? touched : kSlice;
    const float rep = r.of(p.repetition, 1.0f), freq = r.of(p.frequency, 0.0f), pres = r.of(p.presence, 0.0f);
#pragma unroll 1
    for (int i = tid; i < all; i += kAdjustThreads) {
        const int at = touched <= kAdjustList ? (int)list_s[i] : i, v = v0 + at;
        const uint32_t word = adjust_table[at];
        if (!word || !adjust_open(mask, v)) continue;
        r.change(x, y, kType, v, word, p.bias_table ? adjust_table[at + kSlice] : 0u, rep, freq, pres);
    }
}

}  // namespace ws
