// Values of rows as the operators' kernels load and store them: one by one of either type, or eight together.
#pragma once

#include "ws_device.cuh"

namespace ws {

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
    __device__ __forceinline__ void load_all(const void *p, int64_t i) {  // (without the zeros)
        if constexpr (F32)
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(static_cast<const float *>(p) + i) : "memory");
        else
            asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(static_cast<const uint16_t *>(p) + i) : "memory");
    }
    __device__ __forceinline__ float get(int e) const {
        return __uint_as_float(F32 ? w[F32 ? e : 0] : e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    }
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

}  // namespace ws
