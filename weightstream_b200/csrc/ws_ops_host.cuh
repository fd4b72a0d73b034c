// What the C entry points of the operators share: the caller's message buffer, checks of alignment, launches.
#pragma once

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "ws_device.cuh"

namespace ws {

struct Err {  // the caller's message buffer
    char *p;
    size_t len;
    ws_status_t operator()(ws_status_t st, const char *fmt, ...) const {
        if (p && len) {
            va_list ap;
            va_start(ap, fmt);
            vsnprintf(p, len, fmt, ap);
            va_end(ap);
        }
        return st;
    }
};

inline bool is_type(int32_t t) { return t == WS_ACT_BF16 || t == WS_ACT_F32; }
inline int64_t type_bytes(int32_t t) { return t == WS_ACT_BF16 ? 2 : 4; }
inline bool aligned(const void *p, int64_t ld, int32_t type, int64_t bytes) {  // first values of all rows
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * type_bytes(type) % bytes == 0;
}
inline bool natural(const void *p, int32_t type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0; }

// Raises a kernel's limit of dynamic shared memory, once a device.
template <auto K>
ws_status_t allow_smem(const Err &err, int bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (e == cudaSuccess && (device > 63 || !(done.load(std::memory_order_relaxed) & bit))) {
        e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    }
    return e == cudaSuccess ? WS_OK : err(WS_ERR_CUDA, "%d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
}

// The kernels wait for the one before them (griddepcontrol.wait) before they read what it may have written, so their launch
// may overlap its end.  (One of a call's own kernels may read earlier what the call's first one has waited for.)
template <typename P>
ws_status_t launch(const Err &err, void (*kernel)(P), dim3 grid, unsigned threads, size_t smem, unsigned cluster, void *stream, const P &params) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params);
    return e == cudaSuccess ? WS_OK : err(WS_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
}

}  // namespace ws
